// The 8-bit K/V cache: its device layout and the host-side launchers of its kernels (kv8.cu,
// kv8_attn.cu).
//
// A cache holds K and V of `n_seqs` sequences and `heads` K/V heads as signed bytes
//   codes [K|V][seq][head][slot 0 .. cap-1][dim]
//   exps  [K|V][seq][head][slot / 16]
// and a code q of a block of 16 tokens with exponent e stands for q * 2^e, |q| <= 127.  Position p of
// a sequence lives in slot p % cap: the cache is a ring, and a sequence that never passes `cap`
// positions uses it as a plain array.  A scale that is a power of two makes every value exact in
// bf16 and f16 arithmetic, makes the quantisation the same on every machine, and lets a block that
// outgrows its scale be moved to the next one by a rounded shift.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace stt {

constexpr int kKv8Block = 16;       // tokens that share an exponent
constexpr int kKv8MinExp = -100;    // exponent of a block that holds only zeros
constexpr int kKv8Rows = 8;         // query rows of a K/V head that one CTA of the attention takes
constexpr int kKv8MaxPartials = 2048;  // CTAs of one attention call that may leave partial results

enum Dtype : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

struct Kv8Dev {
    int8_t *kc, *vc, *ke, *ve;
    int32_t n_seqs, heads, dim, cap;
    int32_t* err;  // first STT_E_* code that a kernel raised
};

// The batch of a call, device arrays of n entries: sequence (NULL: i), first position, number of
// tokens (NULL: `tokens`).
struct Kv8Batch {
    const int32_t *seqs, *pos, *count;
    int32_t n, tokens;
};

// Rows [n][tokens][heads][dim] with strides in elements, the last dimension contiguous.
struct Kv8Strides {
    int64_t seq, token, head;
};

struct Kv8Attention {
    const void* q;
    void* out;
    Kv8Strides qs, os;
    int32_t q_dtype, out_dtype;
    int32_t group;         // query heads per K/V head
    int32_t window;        // positions that a query sees, its own included; 0: all
    const int32_t* start;  // first position that counts in each sequence of the batch, or NULL
    float scale;
    // workspace: partial results [kKv8MaxPartials][kKv8Rows][dim + 4] and one ticket per merged item
    float* part;
    uint32_t* tickets;
};

size_t kv8_partial_bytes(int dim);

// What the choice between kernels needs to know of a device.
struct Kv8Machine {
    int num_sms;
    int prompt_ctas[4];  // CTAs of the prompt kernel that run at a time, in clusters of 1, 2, 4 and 8
};
cudaError_t kv8_configure(int num_sms, Kv8Machine* m);
cudaError_t launch_kv8_append(const Kv8Dev& c, const Kv8Batch& b, const void* k, const void* v, int dtype,
                              const Kv8Strides& ks, const Kv8Strides& vs, cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8Dev& c, const Kv8Batch& b, void* k, void* v, int dtype, const Kv8Strides& ks,
                            const Kv8Strides& vs, cudaStream_t st);
// The two kernels of the attention: 8 query rows against a split of the keys (any type), and 256 query
// rows on the 5th-generation tensor cores (16-bit queries and output).
struct PromptPlan {
    int cluster;  // CTAs that share a row block's keys
    double us;    // the time that a model gives it
};
PromptPlan kv8_prompt_plan(int64_t rows, int64_t items, int64_t blocks, int out_dtype, const Kv8Machine& m);
cudaError_t launch_kv8_prompt(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, int cluster, cudaStream_t st);
cudaError_t kv8_configure_prompt(Kv8Machine* m);
cudaError_t launch_kv8_attention(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, const Kv8Machine& m,
                                 cudaStream_t st);

}  // namespace stt
