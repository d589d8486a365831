// Host-side internals of libmgprims: the context and the kernel launchers each
// kernel file provides. Launchers validate shapes before they launch and throw
// std::runtime_error; the C ABI turns that into -1 + mg_last_error().
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <stdexcept>
#include <cmath>
#include <string>

#include "mg_softcap_fast.hpp"

struct mg_ctx
{
    int device = 0;
    hipStream_t stream = nullptr; // where every call launches (NULL: the default stream)
    int num_cus = 256;
    // silu/sigmoid of every 16-bit input, as output bits:
    // [0] silu bf16, [1] sigmoid bf16, [2] silu f16, [3] sigmoid f16 (65536 each)
    uint16_t *lut = nullptr;
    void *work = nullptr; // reduction partials (softmax split rows, vocab chunks)
    int64_t work_bytes = 0;
    hipEvent_t handoff = nullptr; // orders a new stream after the old one (mg_set_stream)
};

namespace mg
{
    [[noreturn]] inline void fail(const std::string &m) { throw std::runtime_error(m); }
    inline void check(hipError_t e, const char *what)
    {
        if (e != hipSuccess) fail(std::string(what) + ": " + hipGetErrorString(e));
    }
    inline void check_launch(const char *what) { check(hipGetLastError(), what); }
    // whether a launch takes them: its threads along an axis are counted in 32 bits
    inline bool launchable(int64_t groups, int threads) { return groups <= int64_t(0xffffffff) / threads; }
    inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
    using mgm::recip_rn; // RN(1 / c), mg_softcap_fast.hpp (shared with its host checker)
    inline int dt_size(int dt)
    {
        switch (dt) {
        case 0: return 8;
        case 1: case 2: return 2;
        case 3: return 4;
        default: fail("unknown dtype " + std::to_string(dt));
        }
    }
    inline void need(bool ok, const std::string &m)
    {
        if (!ok) fail(m);
    }

    // log2 of a KV page's tokens: a power of two, so that a position's page and place are a shift and a mask
    inline int page_shift(int64_t page_size, const char *who)
    {
        need(page_size > 0 && page_size <= (int64_t(1) << 20) && (page_size & (page_size - 1)) == 0,
             std::string(who) + ": page_size must be a power of two of at most 2^20 (got " + std::to_string(page_size) + ")");
        return __builtin_ctzll(static_cast<unsigned long long>(page_size));
    }

    // lookup tables, built at mg_open (k_elementwise.hip)
    void build_luts(mg_ctx *c);

    // k_norm.hip
    void launch_norm(mg_ctx *c, int kind, void *h, const void *x, int64_t ldh, int64_t ldx,
                     const void *w, double eps, void *y, int64_t ldy, int64_t rows, int64_t dim,
                     int dt);
    void launch_norm_mixed(mg_ctx *c, int kind, const void *x, int64_t ldx, int dtx, const void *w, int dtw,
                           double eps, void *y, int64_t ldy, int dty, int64_t rows, int64_t dim);
    // k_elementwise.hip
    void launch_residual_add(mg_ctx *c, void *h, const void *x, int64_t n, int dt);
    void launch_swiglu(mg_ctx *c, const void *g, const void *u, void *out, int64_t n, int dt,
                       bool sigmoid_gate);
    void launch_scale(mg_ctx *c, void *x, int64_t n, double s, int dt);
    void launch_softcap(mg_ctx *c, void *z, int64_t n, double mult, double cap, int dt);
    // k_rope.hip
    void launch_rope_table(mg_ctx *c, double theta, int64_t dim, int64_t T, int dt, void *co,
                           void *si);
    void launch_qk_norm_rope(mg_ctx *c, void *q, int64_t nq, int64_t ldq, void *k, int64_t nkv, int64_t ldk,
                             int64_t T, int64_t D, double eps, double qk_scale, const void *co, const void *si,
                             int64_t table_rows, const int64_t *pos, int64_t pos0, const void *v, int64_t ldv,
                             void *kc, void *vc, int64_t slots, int dt);
    void launch_rope(mg_ctx *c, void *q, int64_t qh, int64_t ldq, void *k, int64_t kh,
                     int64_t ldk, int64_t tokens, int64_t dim, const void *co, const void *si,
                     int64_t table_rows, const int64_t *pos, int64_t pos0, int dt);
    // k_softmax.hip
    void launch_softmax(mg_ctx *c, const void *x, int64_t ldx, void *y, int64_t ldy, int64_t heads, int64_t q,
                        int64_t kc, double scale, int mask, int64_t window, int64_t q_pos0, double softcap,
                        int dt_in, int dt_out);
    // k_softmax64.hip (f64 scores: the pure f64 and the f32-compat chains)
    void launch_softmax_f64(mg_ctx *c, const void *x, int64_t ldx, void *y, int64_t ldy, int64_t rows, int64_t q,
                            int64_t kc, double scale, int mask, int64_t window, int64_t q_pos0, double softcap,
                            bool compat);
    // k_q8.hip
    void launch_dequant_q8_0(mg_ctx *c, const int8_t *qs, const uint16_t *d, void *out,
                             int64_t rows, int64_t in, int dt_out);
    // k_vocab.hip
    // mg_npy.cpp (host: .npy files to and from device tensors)
    void npy_info(const char *path, char *descr, int64_t *shape, int max_ndim, int *ndim);
    void npy_load(mg_ctx *c, const char *path, void *dst, int64_t n, int dt);
    void npy_save(mg_ctx *c, const char *path, const void *src, int dt, const int64_t *shape, int ndim);
    void npy_save_i64(mg_ctx *c, const char *path, const int64_t *src, int64_t n);
    // k_sample.hip
    void launch_sample_dist(mg_ctx *c, const int64_t *top_idx, const float *top_val, const int64_t *amax,
                            const int64_t *raw_amax, int64_t rows, int64_t K, double temperature, double top_p,
                            double min_p, int64_t *out_ids, float *out_p, int64_t *out_n);
    void launch_sample_rows(mg_ctx *c, const float *lg, int64_t ld, int64_t rows, int64_t V,
                            const int64_t *raw_amax, int64_t top_k, double temperature, double top_p, double min_p,
                            int64_t *out_ids, float *out_p, int64_t *out_n);
    void launch_quantize_q8_0(mg_ctx *c, const uint16_t *w, int64_t rows, int64_t in, int8_t *qs, uint16_t *d);
    void launch_gemv_q8_0(mg_ctx *c, const int8_t *qs, const uint16_t *d, const uint16_t *x, int64_t batch,
                          int64_t rows, int64_t in, int64_t ldx, float *y, int64_t ldy, bool blockdot);
    void launch_attn_prefill(mg_ctx *c, const uint16_t *q, int64_t ldq, const uint16_t *kc, const uint16_t *vc,
                             int64_t T, int64_t nq, int64_t nkv, int64_t D, int64_t slots, int64_t pos0,
                             int64_t window, double scaling, float *out, int64_t ldo);
    void launch_attn_decode(mg_ctx *c, const uint16_t *q, const uint16_t *kc, const uint16_t *vc, int64_t nq,
                            int64_t nkv, int64_t D, int64_t slots, int64_t qpos, int64_t window, double scaling,
                            float *out);
    // the paged KV cache: k_pages.hip (tables and maps), k_qk.hip (append), k_attn_paged.hip (decode attention)
    void launch_kv_pages(mg_ctx *c, int32_t *table, int64_t ldt, int64_t requests, int64_t max_pages,
                         const int32_t *old_lens, const int32_t *new_lens, int64_t page_size, int32_t *ring,
                         int64_t num_pages, const int64_t *ends, int32_t *lens, int64_t *ends_out, int32_t *starts,
                         int64_t *slots, int64_t *pos, int64_t tokens);
    void launch_qk_norm_rope_paged(mg_ctx *c, void *q, int64_t nq, int64_t ldq, void *k, int64_t nkv, int64_t ldk,
                                   const void *v, int64_t ldv, int64_t T, int64_t D, double eps, double qk_scale,
                                   const void *co, const void *si, int64_t table_rows, const int64_t *pos,
                                   const int64_t *slot_map, void *kc, void *vc, void *kd, void *vd, bool mx,
                                   int64_t slots, int dt);
    void launch_attn_decode_paged(mg_ctx *c, const void *q, int64_t ldq, const void *kc, const void *vc,
                                  const uint16_t *kd, const uint16_t *vd, const int32_t *table, int64_t ldt,
                                  int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq, int64_t nkv,
                                  int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                                  void *out, int64_t ldo, int dt, int dt_out);
    // k_mxfp4.hip
    void launch_quantize_mxfp4(mg_ctx *c, const void *x, int64_t ldx, int64_t rows, int64_t in, int dt, uint8_t *qs,
                               uint8_t *s);
    void launch_dequant_mxfp4(mg_ctx *c, const uint8_t *qs, const uint8_t *s, void *out, int64_t rows, int64_t in,
                              int dt);
    void launch_gemv_mxfp4(mg_ctx *c, const uint8_t *qs, const uint8_t *s, const void *x, int64_t ldx, int64_t batch,
                           int64_t rows, int64_t in, void *y, int64_t ldy, int dt, int dt_out);
    void launch_gemm_mxfp4(mg_ctx *c, const uint8_t *aq, const uint8_t *as, int64_t tokens, const uint8_t *qs,
                           const uint8_t *s, int64_t rows, int64_t in, void *y, int64_t ldy, int dt_out);
    // k_mxfp4_gemm.hip: large products; whether it took the call
    bool launch_mxfp4_tiles(mg_ctx *c, const uint8_t *aq, const uint8_t *as, int64_t tokens, const uint8_t *qs,
                            const uint8_t *s, int64_t rows, int64_t in, void *y, int64_t ldy, int dt_out);
    void join_splits(mg_ctx *c, const float *part, int ns, void *y, int64_t ldy, int64_t rows, int64_t T, int dt_out);
    // k_attn_mxfp4.hip
    void launch_attn_decode_mxfp4(mg_ctx *c, const void *q, int64_t ldq, const uint8_t *kc, const uint8_t *vc,
                                  const uint8_t *ks, const uint8_t *vs, const int32_t *table, int64_t ldt,
                                  int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq, int64_t nkv,
                                  int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                                  void *out, int64_t ldo, int dt, int dt_out);
    void launch_vocab(mg_ctx *c, const void *logits, int64_t ld, int64_t rows, int64_t V, int dt_in, int64_t K,
                      double *lse, int64_t *amax, int64_t *top_idx, float *top_val, bool tail_on, double mult,
                      double cap, void *logits_out);
    // the vocab pass without a context: partials in a fixed device array of
    // kVocabScratchBytes (k_vocab.hip), on `stream` of the current device
    constexpr int64_t kVocabScratchBytes = int64_t(16) << 20;
    // HBM stream probes (k_probe.hip): kind 0 copy, 1 read, 2 write, 3 2r2w
    void launch_probe(mg_ctx *ctx, int kind, void *a, void *b, const void *c, void *d, int64_t bytes);
    void launch_vocab_noalloc(hipStream_t stream, const void *logits, int64_t ld, int64_t rows, int64_t V,
                              int dt_in, int64_t K, double *lse, int64_t *amax, int64_t *top_idx, float *top_val);
} // namespace mg
