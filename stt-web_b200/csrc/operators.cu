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
    int device = 0, num_sms = 0;
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
int beam_tiles(int vocab) { return (vocab + 7 + kBeamChunk - 1) / kBeamChunk; }
int beam_max_chunks(int vocab) { return std::min(kBeamMaxChunks, beam_tiles(vocab)); }

// n_seqs * heads * capacity * dim and the sizes derived from it; false if the arguments do not make a cache.
bool kv8_sizes(int n_seqs, int heads, int dim, int cap, size_t* codes, size_t* exps) {
    if (n_seqs <= 0 || heads <= 0 || (dim != 64 && dim != 128) || cap <= 0 || cap % kKv8Block != 0) return false;
    const unsigned __int128 slots = (unsigned __int128)n_seqs * heads * cap;
    if (slots * dim > (unsigned __int128)1 << 48) return false;
    *codes = (size_t)slots * dim;
    *exps = (size_t)slots / kKv8Block;
    return true;
}

int check_rows(const char* what, const void* p, int dtype, const Kv8Strides& s) {
    const int64_t eb = elem_bytes(dtype);
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || s.seq * eb % 16 != 0 || s.token * eb % 16 != 0 || s.head * eb % 16 != 0)
        return set_error(STT_E_INVALID_ARG, "%s must start at, and have strides of, multiples of 16 bytes", what);
    return STT_OK;
}

int check_batch(const stt_kv8_cache* h, const int32_t* d_seqs, int n, const int32_t* d_pos, int n_tokens, int dtype) {
    if (!h || n < 0 || n_tokens < 0 || (!d_pos && n > 0 && n_tokens > 0)) return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (dtype < DT_F32 || dtype > DT_F16) return set_error(STT_E_INVALID_ARG, "dtype %d unknown", dtype);
    if (!d_seqs && n > h->c.n_seqs)
        return set_error(STT_E_INVALID_ARG, "%d rows for the %d sequences of the cache", n, h->c.n_seqs);
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
    CUDA_TRY(cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device));
    CUDA_TRY(kv8_configure());
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
    return set_error(STT_E_DEVICE_FLAG, "an infinity or NaN was appended to this cache and stored as a finite value");
}

extern "C" int stt_kv8_append_device(stt_kv8_cache* h, const int32_t* d_seqs, int n, const int32_t* d_pos,
                                     const int32_t* d_count, int n_tokens, const void* d_k, const void* d_v, int dtype,
                                     int64_t seq_stride, int64_t token_stride, int64_t head_stride, void* cuda_stream) {
    clear_error();
    TRY(check_batch(h, d_seqs, n, d_pos, n_tokens, dtype));
    if (n == 0 || n_tokens == 0) return STT_OK;
    if (!d_k || !d_v) return set_error(STT_E_INVALID_ARG, "NULL argument");
    if (n_tokens > h->c.cap)
        return set_error(STT_E_INVALID_ARG, "%d tokens in one call exceed the capacity %d", n_tokens, h->c.cap);
    const Kv8Strides s{seq_stride, token_stride, head_stride};
    TRY(check_rows("K", d_k, dtype, s));
    TRY(check_rows("V", d_v, dtype, s));
    if ((int64_t)n * (n_tokens / kKv8Block + 2) > INT_MAX / (h->c.heads + 8))
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", n, n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_append(h->c, Kv8Batch{d_seqs, d_pos, d_count, n, n_tokens}, d_k, d_v, dtype, s,
                               static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_kv8_read_device(const stt_kv8_cache* h, const int32_t* d_seqs, int n, const int32_t* d_pos,
                                   const int32_t* d_count, int n_tokens, void* d_k, void* d_v, int dtype,
                                   int64_t seq_stride, int64_t token_stride, int64_t head_stride, void* cuda_stream) {
    clear_error();
    TRY(check_batch(h, d_seqs, n, d_pos, n_tokens, dtype));
    if (n == 0 || n_tokens == 0) return STT_OK;
    if (!d_k || !d_v) return set_error(STT_E_INVALID_ARG, "NULL argument");
    const Kv8Strides s{seq_stride, token_stride, head_stride};
    TRY(check_rows("K", d_k, dtype, s));
    TRY(check_rows("V", d_v, dtype, s));
    if ((int64_t)n * (n_tokens / 16 + 1) > INT_MAX / (h->c.heads / 8 + 1))
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", n, n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_read(h->c, Kv8Batch{d_seqs, d_pos, d_count, n, n_tokens}, d_k, d_v, dtype, s,
                             static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_kv8_attention_device(stt_kv8_cache* h, const int32_t* d_seqs, int n, const int32_t* d_pos,
                                        const int32_t* d_count, int n_tokens, int n_heads, const void* d_q, int q_dtype,
                                        int64_t q_seq_stride, int64_t q_token_stride, int64_t q_head_stride,
                                        const int32_t* d_start, int window, float scale, void* d_out, int out_dtype,
                                        int64_t out_seq_stride, int64_t out_token_stride, int64_t out_head_stride,
                                        void* cuda_stream) {
    clear_error();
    TRY(check_batch(h, d_seqs, n, d_pos, n_tokens, q_dtype));
    if (window < 0 || !std::isfinite(scale)) return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (out_dtype < DT_F32 || out_dtype > DT_F16) return set_error(STT_E_INVALID_ARG, "dtype %d unknown", out_dtype);
    if (n_heads <= 0 || n_heads % h->c.heads != 0)
        return set_error(STT_E_INVALID_ARG, "%d query heads over %d K/V heads", n_heads, h->c.heads);
    if (n == 0 || n_tokens == 0) return STT_OK;
    if (!d_q || !d_out) return set_error(STT_E_INVALID_ARG, "NULL argument");
    Kv8Attention a{};
    a.q = d_q;
    a.out = d_out;
    a.qs = Kv8Strides{q_seq_stride, q_token_stride, q_head_stride};
    a.os = Kv8Strides{out_seq_stride, out_token_stride, out_head_stride};
    TRY(check_rows("the queries", d_q, q_dtype, a.qs));
    TRY(check_rows("the output", d_out, out_dtype, a.os));
    a.q_dtype = q_dtype;
    a.out_dtype = out_dtype;
    a.group = n_heads / h->c.heads;
    a.window = window;
    a.start = d_start;
    a.scale = scale;
    a.part = h->part;
    a.tickets = h->tickets;
    a.num_sms = h->num_sms;
    const int64_t row_groups = ((int64_t)n_tokens * a.group + kKv8Rows - 1) / kKv8Rows;
    if ((int64_t)n_tokens * a.group > INT_MAX - kKv8Rows || (int64_t)n * h->c.heads > INT_MAX / row_groups)
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", n, n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_attention(h->c, Kv8Batch{d_seqs, d_pos, d_count, n, n_tokens}, a,
                                  static_cast<cudaStream_t>(cuda_stream)));
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
    if ((int64_t)max_beams * max_vocab > INT_MAX - kBeamChunk || (int64_t)max_batch * max_beams * beam_max_chunks(max_vocab) > INT_MAX)
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
    const size_t parts = (size_t)max_batch * max_beams * beam_max_chunks(max_vocab);
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
    return set_error(STT_E_DEVICE_FLAG, "a beam had a NaN or +inf logit or score: its candidates were taken as -inf");
}

extern "C" int stt_beam_select_device(stt_beam* h, const void* d_logits, int dtype, int64_t row_stride, int batch,
                                      int beams, int vocab, const float* d_scores, const uint8_t* d_done, int eos,
                                      float* d_next_scores, int32_t* d_parents, int32_t* d_tokens, uint8_t* d_next_done,
                                      void* cuda_stream) {
    clear_error();
    if (!h || batch < 0 || (batch > 0 && (!d_logits || !d_scores || !d_next_scores || !d_parents || !d_tokens)))
        return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (dtype < DT_F32 || dtype > DT_F16) return set_error(STT_E_INVALID_ARG, "dtype %d unknown", dtype);
    if (beams < 1 || vocab < 1 || !beam_fits(h, batch, beams, vocab))
        return set_error(STT_E_INVALID_ARG, "%d utterances, %d beams, %d tokens: the selector was made for %d, %d, %d", batch,
                         beams, vocab, h->max_batch, h->max_beams, h->max_vocab);
    if (row_stride < vocab) return set_error(STT_E_INVALID_ARG, "row stride %lld < vocab %d", (long long)row_stride, vocab);
    if (eos < -1 || eos >= vocab) return set_error(STT_E_INVALID_ARG, "end token %d outside the %d tokens", eos, vocab);
    if (d_done && eos < 0) return set_error(STT_E_INVALID_ARG, "beams that ended need an end token");
    if (reinterpret_cast<uintptr_t>(d_logits) % elem_bytes(dtype) != 0)
        return set_error(STT_E_INVALID_ARG, "the logits must be aligned to their type");
    if (batch == 0) return STT_OK;
    BeamArgs a = h->ws;
    a.logits = d_logits;
    a.row_stride = row_stride;
    a.batch = batch;
    a.beams = beams;
    a.vocab = vocab;
    // about four CTAs per SM, twice what is resident (rows that ended leave gaps); a CTA takes whole tiles
    const int tiles = beam_tiles(vocab), rows = batch * beams;
    const int want = std::min(beam_max_chunks(vocab), (4 * h->num_sms + rows - 1) / rows);
    a.tiles_per_chunk = (tiles + want - 1) / want;
    a.chunks = (tiles + a.tiles_per_chunk - 1) / a.tiles_per_chunk;
    a.scores = d_scores;
    a.done = d_done;
    a.eos = eos;
    a.next_scores = d_next_scores;
    a.parents = d_parents;
    a.tokens = d_tokens;
    a.next_done = d_next_done;
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_beam_select(a, dtype, static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_beam_reorder_device(int device, void* d_states, int64_t row_stride, int segments,
                                       int64_t segment_stride, int64_t units, int64_t unit_bytes,
                                       const int32_t* d_parents, int groups, int beams, const int32_t* d_held,
                                       void* cuda_stream) {
    clear_error();
    if (!d_states || !d_parents || segments < 0 || units < 0 || unit_bytes <= 0 || groups < 0)
        return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (beams < 1 || beams > kMaxBeams) return set_error(STT_E_INVALID_ARG, "beams %d out of range [1, %d]", beams, kMaxBeams);
    const __int128 segment = (__int128)units * unit_bytes;
    if (segment > (__int128)1 << 38) return set_error(STT_E_INVALID_ARG, "segments of %lld x %lld bytes are too large", (long long)units, (long long)unit_bytes);
    // rows and segments must not overlap: a position belongs to one of them
    if ((segments > 1 && segment_stride < segment) || (groups * (int64_t)beams > 1 && row_stride < 0))
        return set_error(STT_E_INVALID_ARG, "segments overlap");
    const __int128 row = segments == 0 ? 0 : (__int128)(segments - 1) * segment_stride + segment;
    const bool interleaved = (int64_t)groups * beams > 1 && row_stride < row;
    if (interleaved && !(row_stride >= segment && segment_stride >= (__int128)row_stride * ((int64_t)groups * beams - 1) + segment))
        return set_error(STT_E_INVALID_ARG, "rows overlap");
    DeviceScope ds(device);
    if (!ds.ok) {
        (void)cudaGetLastError();
        return set_error(STT_E_INVALID_ARG, "cannot select device %d", device);
    }
    ReorderArgs a{};
    a.states = static_cast<uint8_t*>(d_states);
    a.row_stride = row_stride;
    a.segment_stride = segment_stride;
    a.inner = std::max(1, segments);
    a.per_unit = 1;
    a.units = units;
    a.unit_bytes = unit_bytes;
    a.segments = segments;
    a.groups = groups;
    a.beams = beams;
    a.parents = d_parents;
    a.held = d_held;
    CUDA_TRY(launch_reorder(a, static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}
