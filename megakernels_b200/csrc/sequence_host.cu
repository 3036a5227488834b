// C ABI of libmkb200_sequences.so (declared in include/mkb200_sequences.h): the checks of arguments, then the launches.
#include <cstdarg>
#include <cstdio>

#include "sequence_kernels.h"

namespace {

thread_local char g_error[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}
int invalid(const char* what) { return fail(MKBS_ERR_INVALID_ARGUMENT, "%s", what); }

bool aligned(const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; }

int launched(const char* what, cudaError_t e) {
    return e == cudaSuccess ? (int)MKBS_OK : fail(MKBS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// The library's code is for one architecture.
int check_device() {
    static thread_local int known = -1;
    int dev = 0, major = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev == known) return MKBS_OK;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e != cudaSuccess) return launched("device", e);
    if (major < 10) return fail(MKBS_ERR_UNSUPPORTED, "this library is built for sm_100a only");
    known = dev;
    return MKBS_OK;
}

// What mkb_beam_bytes needs to be right.
int check_shape(const MkbsBeams* b) {
    if (!b || b->struct_bytes != sizeof(MkbsBeams)) return invalid("beams: NULL or another struct size");
    if (b->dtype != MKBS_BF16 && b->dtype != MKBS_F32) return invalid("beams: dtype is bf16 or float");
    if (b->groups < 1 || b->beams < 1 || b->vocab < 1 || b->k < 1) return invalid("beams: groups, beams, vocab and k must be positive");
    if (b->beams > MKBS_MAX_BEAMS || b->k > MKBS_MAX_BEST || (int64_t)b->groups * b->beams > 65535)
        return fail(MKBS_ERR_UNSUPPORTED, "beams: at most %d beams a group, %d best and 65535 rows", MKBS_MAX_BEAMS, MKBS_MAX_BEST);
    if ((int64_t)b->beams * b->vocab > MKBS_MAX_BEAM_WORK / b->k)
        return fail(MKBS_ERR_UNSUPPORTED, "beams: beams * vocab * k above %d", MKBS_MAX_BEAM_WORK);
    if (b->k > (int64_t)b->beams * b->vocab) return invalid("beams: k is more than there are continuations");
    if (mkbs::beam_bytes(*b) == 0) return fail(MKBS_ERR_UNSUPPORTED, "beams: more candidates than shared memory holds");
    return MKBS_OK;
}
int check(const MkbsBeams* b) {
    if (const int rc = check_shape(b)) return rc;
    const uintptr_t elem = b->dtype == MKBS_BF16 ? 2 : 4;
    if (b->row_stride < b->vocab) return invalid("beams: row_stride is less than vocab");
    if (!aligned(b->logits, elem)) return invalid("beams: logits missing or not aligned to their type");
    if ((b->scores && !aligned(b->scores, 4)) || !aligned(b->out_scores, 4) || !aligned(b->out_parents, 4) || !aligned(b->out_tokens, 4))
        return invalid("beams: scores or outputs missing or unaligned");
    if (b->eos < -1 || b->eos >= b->vocab || (b->done && b->eos < 0)) return invalid("beams: eos outside the vocabulary (-1: none, without done)");
    if (!aligned(b->workspace, 16) || b->workspace_bytes < mkbs::beam_bytes(*b)) return invalid("beams: workspace missing, unaligned or too small");
    return MKBS_OK;
}

int check(const MkbsReorder* r) {
    if (!r || r->struct_bytes != sizeof(MkbsReorder)) return invalid("reorder: NULL or another struct size");
    if (r->slots < 1 || r->num_regions < 1 || r->first < 0 || !r->regions) return invalid("reorder: slots and regions must be positive, first not negative");
    if (r->slots > MKBS_MAX_SLOTS || r->num_regions > MKBS_MAX_REGIONS)
        return fail(MKBS_ERR_UNSUPPORTED, "reorder: at most %d slots and %d regions", MKBS_MAX_SLOTS, MKBS_MAX_REGIONS);
    if (!aligned(r->parents, 4) || (r->lengths && !aligned(r->lengths, 4)) || (r->status && !aligned(r->status, 4)))
        return invalid("reorder: parents missing, or they, lengths or status unaligned");
    for (int i = 0; i < r->num_regions; ++i) {
        const MkbsRegion& g = r->regions[i];
        if (!g.base || g.outer < 1 || g.rows < 1 || g.row_bytes < 1) return fail(MKBS_ERR_INVALID_ARGUMENT, "reorder: region %d is empty", i);
        if (g.row_bytes > (1 << 30) || g.slot_stride < g.rows * g.row_bytes || !mkbs::apart(g.rows * g.row_bytes, {{g.outer, g.outer_stride}, {r->slots, g.slot_stride}}))
            return fail(MKBS_ERR_INVALID_ARGUMENT, "reorder: slots or layers of region %d overlap", i);
        for (int j = 0; j < i; ++j)  // (blocks would move the same rows at once)
            if (r->regions[j].base == g.base) return fail(MKBS_ERR_INVALID_ARGUMENT, "reorder: regions %d and %d are the same", j, i);
    }
    return MKBS_OK;
}

int check_items(const char* what, int layers, int sequences, int kv_heads, int positions, int length, const void* lengths) {
    if (layers < 1 || sequences < 1 || kv_heads < 1 || positions < 1)
        return fail(MKBS_ERR_INVALID_ARGUMENT, "%s: layers, sequences, heads and positions must be positive", what);
    if (layers > 65535 || sequences > 65535 || kv_heads > 32767 || (int64_t)layers * sequences * kv_heads > 65535)
        return fail(MKBS_ERR_UNSUPPORTED, "%s: more than 65535 layers * sequences * heads", what);
    if (positions > 1 << 28) return fail(MKBS_ERR_UNSUPPORTED, "%s: more than 2^28 positions", what);
    if (lengths ? !aligned(lengths, 4) : length < 0 || length > positions)
        return fail(MKBS_ERR_INVALID_ARGUMENT, "%s: length outside the cache, or unaligned lengths", what);
    return MKBS_OK;
}

int check_shape(const MkbsKeyWeights* w) {
    if (!w || w->struct_bytes != sizeof(MkbsKeyWeights)) return invalid("key weights: NULL or another struct size");
    if (const int rc = check_items("key weights", w->layers, w->sequences, w->kv_heads, w->positions, w->length, w->lengths)) return rc;
    if (w->queries < 1 || w->heads < w->kv_heads || w->heads % w->kv_heads) return invalid("key weights: queries must be positive, heads a multiple of kv_heads");
    if ((w->dim != 64 && w->dim != 128) || w->heads / w->kv_heads > 128 || (int64_t)w->queries * (w->heads / w->kv_heads) > 1 << 20)
        return fail(MKBS_ERR_UNSUPPORTED, "key weights: dim 64 or 128, at most 128 heads of a key and 2^20 queries times them");
    if ((int64_t)w->layers * w->sequences * w->kv_heads * ((w->positions + 127) / 128) > 1 << 30)  // (units of work are counted in 32 bits)
        return fail(MKBS_ERR_UNSUPPORTED, "key weights: more than 2^30 tiles of 128 keys");
    return MKBS_OK;
}
int check(const MkbsKeyWeights* w) {
    if (const int rc = check_shape(w)) return rc;
    const int64_t q_row = (int64_t)w->heads * w->dim, k_row = (int64_t)w->kv_heads * w->dim;
    if (!aligned(w->q, 16) || !aligned(w->k, 16) || !aligned(w->weights, 4) || (w->status && !aligned(w->status, 4)))
        return invalid("key weights: q, k or weights missing or unaligned");
    if ((w->layers > 1 && (w->q_layer % 8 || w->k_layer % 8)) || (w->sequences > 1 && (w->q_sequence % 8 || w->k_sequence % 8)))
        return invalid("key weights: strides of q and k are multiples of 8");
    if ((w->layers > 1 && (w->q_layer < w->queries * q_row || w->k_layer < w->positions * k_row)) ||
        (w->sequences > 1 && (w->q_sequence < w->queries * q_row || w->k_sequence < w->positions * k_row)))
        return invalid("key weights: sequences or layers of q or k overlap");
    if (!mkbs::apart(w->positions, {{w->layers, w->w_layer}, {w->sequences, w->w_sequence}, {w->kv_heads, w->w_head}})) return invalid("key weights: weights overlap");
    if (!(w->scale - w->scale == 0.f)) return invalid("key weights: scale is not finite");
    if (!aligned(w->workspace, 256) || w->workspace_bytes < mkbs::key_weights_bytes(*w))
        return invalid("key weights: workspace missing, unaligned or too small");
    return MKBS_OK;
}

int check(const MkbsSelect* s) {
    if (!s || s->struct_bytes != sizeof(MkbsSelect)) return invalid("select: NULL or another struct size");
    if (const int rc = check_items("select", s->layers, s->sequences, s->kv_heads, s->positions, s->length, s->lengths)) return rc;
    if (s->keep < 1 || s->sinks < 0 || s->recent < 0 || (int64_t)s->sinks + s->recent > s->keep)
        return invalid("select: keep must be positive and hold the sinks and the recent rows");
    if (!aligned(s->weights, 4) || !aligned(s->rows, 4) || (s->kept && !aligned(s->kept, 4))) return invalid("select: weights or rows missing or unaligned");
    if (s->kept && !mkbs::apart(s->positions, {{s->layers, s->w_layer}, {s->sequences, s->w_sequence}, {s->kv_heads, s->w_head}}))
        return invalid("select: kept weights overlap");
    return MKBS_OK;
}

int check(const MkbsMove* m) {
    if (!m || m->struct_bytes != sizeof(MkbsMove)) return invalid("move: NULL or another struct size");
    if (const int rc = check_items("move", m->layers, m->sequences, m->kv_heads, m->positions, m->length, m->lengths)) return rc;
    if (m->keep < 1) return invalid("move: keep must be positive");
    if (m->head_bytes < 16 || m->head_bytes % 16 || m->head_bytes > 1024)
        return fail(MKBS_ERR_UNSUPPORTED, "move: a head's part of a row is a multiple of 16 bytes, at most 1024");
    if (!aligned(m->rows, 4) || !aligned(m->caches[0], 16) || (m->caches[1] && !aligned(m->caches[1], 16)) || (m->layers > 1 && m->c_layer % 16) ||
        (m->sequences > 1 && m->c_sequence % 16))
        return invalid("move: rows or caches missing or unaligned");
    if (m->caches[0] == m->caches[1]) return invalid("move: both caches are the same");
    if (!mkbs::apart((int64_t)m->positions * m->kv_heads * m->head_bytes, {{m->layers, m->c_layer}, {m->sequences, m->c_sequence}}))
        return invalid("move: sequences or layers overlap");
    return MKBS_OK;
}

}  // namespace

extern "C" {

size_t mkb_beam_bytes(const MkbsBeams* b) { return check_shape(b) ? 0 : mkbs::beam_bytes(*b); }
int mkb_beam_select(const MkbsBeams* b, void* stream) {
    if (int rc = check(b); rc || (rc = check_device())) return rc;
    return launched("beams", mkbs::beam_launch(*b, static_cast<cudaStream_t>(stream)));
}
int mkb_reorder_slots(const MkbsReorder* r, void* stream) {
    if (int rc = check(r); rc || (rc = check_device())) return rc;
    return launched("reorder", mkbs::reorder_launch(*r, static_cast<cudaStream_t>(stream)));
}
size_t mkb_key_weights_bytes(const MkbsKeyWeights* w) { return check_shape(w) ? 0 : mkbs::key_weights_bytes(*w); }
int mkb_key_weights(const MkbsKeyWeights* w, void* stream) {
    if (int rc = check(w); rc || (rc = check_device())) return rc;
    return launched("key weights", mkbs::key_weights_launch(*w, static_cast<cudaStream_t>(stream)));
}
int mkb_select_rows(const MkbsSelect* s, void* stream) {
    if (int rc = check(s); rc || (rc = check_device())) return rc;
    return launched("select", mkbs::select_launch(*s, static_cast<cudaStream_t>(stream)));
}
int mkb_move_rows(const MkbsMove* m, void* stream) {
    if (int rc = check(m); rc || (rc = check_device())) return rc;
    return launched("move", mkbs::move_launch(*m, static_cast<cudaStream_t>(stream)));
}
const char* mkb_sequences_last_error(void) { return g_error; }
int mkb_sequences_abi_version(void) { return MKBS_ABI_VERSION; }
size_t mkb_sequences_struct_bytes(int32_t which) {
    const size_t sizes[] = {sizeof(MkbsBeams), sizeof(MkbsRegion), sizeof(MkbsReorder), sizeof(MkbsKeyWeights), sizeof(MkbsSelect), sizeof(MkbsMove)};
    return which >= 0 && which < 6 ? sizes[which] : 0;
}

}  // extern "C"
