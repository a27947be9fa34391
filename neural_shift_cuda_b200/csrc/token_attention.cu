// token_attention.cu -- C entry points of token attention: argument checks and
// the choice of kernel family.
#include <climits>

#include "token_attention.h"

namespace nsc {
namespace tok {
namespace {

nsc_status check(const char* op, const nsc_attention* a, bool need_ptrs) {
    if (!a) return fail(NSC_ERR_INVALID_ARG, "%s: arguments are NULL", op);
    if (!valid_dtype(a->dtype))
        return fail(NSC_ERR_UNSUPPORTED_DTYPE, "%s: unsupported dtype code %d", op, a->dtype);
    if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->Hq < 1 || a->Hkv < 1 || a->D < 1)
        return fail(NSC_ERR_INVALID_ARG, "%s: bad extent", op);
    if (a->Hq % a->Hkv)
        return fail(NSC_ERR_INVALID_ARG,
                    "%s: %lld query heads are not a multiple of %lld key heads", op,
                    (long long)a->Hq, (long long)a->Hkv);
    const int64_t widest = a->dtype == NSC_F64 ? 128 : 256;
    if (a->D > widest)
        return fail(NSC_ERR_INVALID_ARG, "%s: head width %lld exceeds %lld", op, (long long)a->D,
                    (long long)widest);
    // positions and tile counts are 32-bit; offsets are 64-bit
    if (a->Lq >= (1LL << 30) || a->Lk >= (1LL << 30) || a->Hq >= (1LL << 16) ||
        a->B * a->Hq >= (1LL << 31) / ((a->Lq > a->Lk ? a->Lq : a->Lk) / 32 + 2))
        return fail(NSC_ERR_INVALID_ARG, "%s: too many tokens", op);
    if (!(a->softcap >= 0) || a->softcap > 1e30 || (a->softcap > 0 && a->softcap < 1e-30))
        return fail(NSC_ERR_INVALID_ARG, "%s: softcap must be 0 or in 1e-30..1e30", op);
    if (a->documents && (a->docs < 1 || a->Lq != a->Lk))
        return fail(NSC_ERR_INVALID_ARG, "%s: documents need at least two bounds and Lq == Lk", op);
    if (a->prefix && !a->causal)
        return fail(NSC_ERR_INVALID_ARG, "%s: a prefix needs causal", op);
    if ((a->table != nullptr) != (a->buckets != nullptr))
        return fail(NSC_ERR_INVALID_ARG, "%s: a bias needs its table and its buckets", op);
    if (a->table) {
        if (a->n_buckets < 1 || a->n_buckets > 256 || a->reach < 0 || a->reach > 1024)
            return fail(NSC_ERR_INVALID_ARG,
                        "%s: a bias has 1..256 buckets and a reach of 0..1024 (got %lld, %lld)",
                        op, (long long)a->n_buckets, (long long)a->reach);
        const bool half = a->dtype == NSC_F16 || a->dtype == NSC_BF16;
        if (a->table_dtype != a->dtype && !(half && a->table_dtype == NSC_F32))
            return fail(NSC_ERR_UNSUPPORTED_DTYPE,
                        "%s: the bias table has the dtype of q, or fp32 with fp16 / bf16", op);
    }
    if (need_ptrs && a->B && a->Lq && !a->q)
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    if (need_ptrs && a->B && a->Lk && (!a->k || !a->v))
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    return ok();
}

Params params(const nsc_attention* a) {
    Params p{};
    p.q = a->q; p.k = a->k; p.v = a->v;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_stride[i];
        p.ks[i] = a->k_stride[i];
        p.vs[i] = a->v_stride[i];
    }
    p.B = static_cast<int>(a->B);
    p.Lq = static_cast<int>(a->Lq);
    p.Lk = static_cast<int>(a->Lk);
    p.Hq = static_cast<int>(a->Hq);
    p.Hkv = static_cast<int>(a->Hkv);
    p.G = p.Hq / p.Hkv;
    p.D = static_cast<int>(a->D);
    p.causal = a->causal != 0;
    p.docs = a->documents;
    p.n_docs = static_cast<int>(a->docs);
    p.docs_stride = a->docs_stride;
    p.prefix = a->prefix;
    p.prefix_stride = a->prefix_stride;
    p.lengths = a->lengths;
    p.lut = a->buckets;
    p.table = a->table;
    p.table_dtype = a->table_dtype;
    p.nb = static_cast<int>(a->n_buckets);
    p.reach = static_cast<int>(a->reach);
    p.scale = a->scale;
    p.cap = a->softcap;
    return p;
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
bool aligned256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255) == 0; }
int64_t acc_size(int dtype) { return dtype == NSC_F64 ? 8 : 4; }

int query_parts(const nsc_attention* a) {
    const int tl = general_tile(a->dtype, a->B, a->Hkv, a->Lq, a->Lk, a->D);
    return static_cast<int>(a->B * ((a->Lq + tl - 1) / tl));
}

}  // namespace
}  // namespace tok
}  // namespace nsc

using namespace nsc;
using namespace nsc::tok;

extern "C" NSC_API nsc_status nsc_token_attention_fwd(const nsc_attention* a, void* out, void* lse,
                                                      void* stats, void* residue, void* stream) {
    const char* op = "token_attention";
    nsc_status st = check(op, a, true);
    if (st != NSC_OK) return st;
    if (a->lengths)
        return fail(NSC_ERR_INVALID_ARG, "%s: lengths belong to the decode form", op);
    if (!a->B || !a->Lq) return ok();
    if (!out) return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    Params p = params(a);
    p.out = out;
    p.lse = lse;
    p.stats = stats;
    p.residue = residue;
    if (short_fits(p, a->dtype)) return short_fwd(p, a->dtype, as_stream(stream));
    if (tc_fits(p, a->dtype)) return tc_fwd(p, a->dtype, as_stream(stream));
    return general_fwd(p, a->dtype, as_stream(stream));
}

extern "C" NSC_API int64_t nsc_token_attention_bwd_workspace(const nsc_attention* a) {
    if (check("token_attention", a, false) != NSC_OK) return -1;
    int64_t n = align256(a->B * a->Hq * a->Lq * acc_size(a->dtype));
    if (a->table) n += align256(a->Hq * query_parts(a) * a->n_buckets * acc_size(a->dtype));
    // whichever kernels the call will take
    const int64_t tc =
        tc_bwd_workspace(a->B, a->Hq, a->Hkv, a->Lq, a->Lk, a->table ? a->n_buckets : 0);
    return n > tc ? n : tc;
}

extern "C" NSC_API nsc_status nsc_token_attention_bwd(const nsc_attention* a,
                                                      const nsc_attention_grad* g, void* stream) {
    const char* op = "token_attention backward";
    nsc_status st = check(op, a, true);
    if (st != NSC_OK) return st;
    if (!g) return fail(NSC_ERR_INVALID_ARG, "%s: arguments are NULL", op);
    if (a->lengths)
        return fail(NSC_ERR_INVALID_ARG, "%s: lengths belong to the decode form", op);
    const bool rows = a->B && a->Lq, cols = a->B && a->Lk;
    // grad_q comes with grad_table, grad_k with grad_v; a pair that is not wanted is left out
    if ((rows && (!g->out || !g->stats || !g->grad_out || !g->workspace ||
                  (g->grad_table && !g->grad_q))) ||
        (cols && !g->grad_k != !g->grad_v) || (g->grad_table && !a->table))
        return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    if (!aligned256(g->workspace))
        return fail(NSC_ERR_INVALID_ARG, "%s: workspace is not 256-byte aligned", op);
    cudaStream_t s = as_stream(stream);
    Params p = params(a);
    p.out = const_cast<void*>(g->out);
    p.stats = const_cast<void*>(g->stats);
    p.residue = const_cast<void*>(g->residue);
    Grads gr{};
    gr.dout = g->grad_out;
    gr.dlse = g->grad_lse;
    for (int i = 0; i < 3; ++i) gr.dos[i] = g->grad_out_stride[i];
    gr.dq = g->grad_q;
    gr.dk = g->grad_k;
    gr.dv = g->grad_v;
    if (!a->B)   // no rows and no keys; a table's gradient is a sum of nothing
        return g->grad_table ? launch_table_join(p, gr, g->grad_table, s) : ok();
    if (tc_bwd_fits(p, gr, a->dtype))
        return tc_bwd(p, gr, g->workspace, g->grad_table, a->dtype, s);
    gr.delta = g->workspace;
    if (g->grad_table) {
        gr.n_part = rows ? query_parts(a) : 0;
        gr.tab = static_cast<char*>(g->workspace) +
                 align256(a->B * a->Hq * a->Lq * acc_size(a->dtype));
    }
    st = launch_delta(p, gr, a->dtype, s);
    if (st == NSC_OK) st = general_bwd(p, gr, a->dtype, s);
    if (st == NSC_OK && g->grad_table) st = launch_table_join(p, gr, g->grad_table, s);
    return st;
}

extern "C" NSC_API int64_t nsc_token_attention_decode_workspace(const nsc_attention* a) {
    if (check("token_attention_decode", a, false) != NSC_OK) return -1;
    return decode_workspace(params(a), a->dtype);
}

extern "C" NSC_API nsc_status nsc_token_attention_decode(const nsc_attention* a, void* out,
                                                         void* lse, void* workspace,
                                                         void* stream) {
    const char* op = "token_attention_decode";
    nsc_status st = check(op, a, true);
    if (st != NSC_OK) return st;
    if (!a->B || !a->Lq) return ok();
    if (!out) return fail(NSC_ERR_INVALID_ARG, "%s: NULL pointer", op);
    if (a->documents || a->prefix || (a->table && !a->causal))
        return fail(NSC_ERR_INVALID_ARG,
                    "%s: without documents or prefix, and causal with a bias", op);
    if (!aligned256(workspace))
        return fail(NSC_ERR_INVALID_ARG, "%s: workspace is not 256-byte aligned", op);
    Params p = params(a);
    p.out = out;
    p.lse = lse;
    return decode(p, workspace, a->dtype, as_stream(stream));
}
