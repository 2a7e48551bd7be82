/*
 * Gated linear recurrence entry points (kmamba_b200.h): argument checks,
 * sizes, the workspace, and the launches.  No counterpart in the reference,
 * whose recurrences are the selective scans.
 */
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../kmb_internal.h"

static int misaligned(const void *p, size_t n) { return p && ((uintptr_t)p & (n - 1)) != 0; }

static int sizes_ok(const KmbGLR *a) {
    const long lim = 1L << 31;
    return a && a->batch >= 0 && a->L >= 0 && a->D > 0 && a->batch < lim && a->D < lim &&
           a->L < lim * 32 && (a->offsets || a->batch == 0 || a->L < lim * 32 / a->batch);
}

long kmb_glr_ckpt_elems(const KmbGLR *a) {
    if (!sizes_ok(a)) return 0;
    const long chunk = KMB_GLR_CHUNK(a->type), chunks = (a->L + chunk - 1) / chunk;
    return (a->offsets ? 1 : a->batch) * chunks * a->D;
}

size_t kmb_glr_workspace_bytes(const KmbGLR *a, int bwd) {
    if (!sizes_ok(a)) return 0;
    const size_t f = kmb_glr_scratch_bytes(a, 0), b = bwd ? kmb_glr_scratch_bytes(a, 1) : 0;
    return f > b ? f : b; /* one workspace serves a forward and its backward */
}

static int check_rows(const KmbGLR *a, const KmbRows *r, const char *name, int out) {
    const size_t es = a->type == KMB_BF16 ? 2 : 4;
    if (!r->data) return kmb_fail(KMB_EINVAL, "glr: %s is required", name);
    if (misaligned(r->data, es)) return kmb_fail(KMB_EINVAL, "glr: %s is not aligned to its element", name);
    if (r->row_stride < a->D) return kmb_fail(KMB_EINVAL, "glr: row stride of %s smaller than the row", name);
    if (a->offsets || a->batch <= 1) return KMB_OK;
    if (r->batch_stride < a->D)
        return kmb_fail(KMB_EINVAL, "glr: batch stride of %s smaller than the row", name);
    /* rows of different sequences may not share memory in an output:
     * batch-major or time-major */
    if (out && a->L > 1 && r->batch_stride < (a->L - 1) * r->row_stride + a->D &&
        r->row_stride < (a->batch - 1) * r->batch_stride + a->D)
        return kmb_fail(KMB_EINVAL, "glr: the strides of %s make its rows overlap", name);
    return KMB_OK;
}

/* An output may be an input, the very same rows, but not another output. */
static int check_overlap(const KmbGLR *a, const KmbRows *const *in, int ni, const KmbRows *const *out, int no) {
    for (int i = 0; i < no; ++i) {
        for (int j = 0; j < i; ++j)
            if (out[i]->data == out[j]->data) return kmb_fail(KMB_EINVAL, "glr: two outputs share their memory");
        for (int j = 0; j < ni; ++j) {
            if (out[i]->data != in[j]->data) continue;
            if (out[i]->row_stride != in[j]->row_stride ||
                (!a->offsets && a->batch > 1 && out[i]->batch_stride != in[j]->batch_stride))
                return kmb_fail(KMB_EINVAL, "glr: an output over an input of other strides");
        }
    }
    return KMB_OK;
}

static int validate(const KmbGLR *a, int bwd) {
    if (!a) return kmb_fail(KMB_EINVAL, "glr: NULL arguments");
    if (a->batch < 0 || a->L < 0 || a->D <= 0)
        return kmb_fail(KMB_EINVAL, "glr: sizes must be positive");
    if (!sizes_ok(a)) return kmb_fail(KMB_EUNSUPPORTED, "glr: sizes too large");
    if (a->type != KMB_F32 && a->type != KMB_BF16) return kmb_fail(KMB_EINVAL, "glr: unknown element type");
    if (!(a->scale > 0.f) || isinf(a->scale))
        return kmb_fail(KMB_EINVAL, "glr: scale must be positive and finite");
    if (a->accumulate != 0 && a->accumulate != 1)
        return kmb_fail(KMB_EINVAL, "glr: accumulate must be 0 or 1");
    if (!a->decay) return kmb_fail(KMB_EINVAL, "glr: decay is required");
    if (misaligned(a->offsets, 8)) return kmb_fail(KMB_EINVAL, "glr: offsets are not 8-byte aligned");
    const void *f32[] = {a->decay, a->h0, a->h_last, a->ckpt, a->dh_last, a->dh0, a->ddecay};
    for (size_t i = 0; i < sizeof f32 / sizeof *f32; ++i)
        if (misaligned(f32[i], 4)) return kmb_fail(KMB_EINVAL, "glr: an fp32 tensor is not 4-byte aligned");
    if (a->batch == 0 || a->L == 0) return KMB_OK;
    int rc = check_rows(a, &a->x, "x", 0);
    if (!rc) rc = check_rows(a, &a->gate_r, "gate_r", 0);
    if (!rc) rc = check_rows(a, &a->gate_i, "gate_i", 0);
    const KmbRows *in[] = {&a->x, &a->gate_r, &a->gate_i, &a->dy};
    const KmbRows *fwd_out[] = {&a->y}, *bwd_out[] = {&a->dx, &a->dgate_r, &a->dgate_i};
    if (!bwd) {
        if (!rc) rc = check_rows(a, &a->y, "y", 1);
        return rc ? rc : check_overlap(a, in, 3, fwd_out, 1);
    }
    if (!rc) rc = check_rows(a, &a->dy, "dy", 0);
    if (!rc) rc = check_rows(a, &a->dx, "dx", 1);
    if (!rc) rc = check_rows(a, &a->dgate_r, "dgate_r", 1);
    if (!rc) rc = check_rows(a, &a->dgate_i, "dgate_i", 1);
    return rc ? rc : check_overlap(a, in, 4, bwd_out, 3);
}

static int run(const KmbGLR *a, int bwd) {
    KmbStage st;
    KmbGLR d;
    int rc = validate(a, bwd);
    if (rc) return rc;
    const size_t need = kmb_glr_scratch_bytes(a, bwd);
    if (need && a->workspace) {
        if (a->workspace_bytes < need)
            return kmb_fail(KMB_EINVAL, "glr: workspace of %zu bytes, %zu needed", a->workspace_bytes,
                            need);
        if (misaligned(a->workspace, 16))
            return kmb_fail(KMB_EINVAL, "glr: workspace must be 16-byte aligned");
    }
    const void *ws = need ? a->workspace : NULL;
    const void *fwd_ptrs[] = {a->x.data, a->gate_r.data, a->gate_i.data, a->y.data, a->decay,
                              a->h0,     a->h_last,      a->ckpt,        a->offsets, ws};
    const void *bwd_ptrs[] = {a->x.data,  a->gate_r.data,  a->gate_i.data,  a->dy.data,
                              a->dx.data, a->dgate_r.data, a->dgate_i.data, a->decay,
                              a->h0,      a->ckpt,         a->dh_last,      a->dh0,
                              a->ddecay,  a->offsets,      ws};
    rc = bwd ? kmb_check_device_ptrs("glr", bwd_ptrs, sizeof bwd_ptrs / sizeof *bwd_ptrs)
             : kmb_check_device_ptrs("glr", fwd_ptrs, sizeof fwd_ptrs / sizeof *fwd_ptrs);
    if (rc) return rc;
    if ((rc = kmb_check_capture("glr", kmb_stream(), need && !a->workspace))) return rc;
    kmb_stage_begin(&st);
    d = *a;
    if (need && !d.workspace) d.workspace = kmb_scratch(&st, need);
    rc = st.status;
    if (!rc) rc = bwd ? kmb_launch_glr_bwd(&d, st.s) : kmb_launch_glr_fwd(&d, st.s);
    rc = kmb_stage_finish(&st, rc);
    return !rc && need && kmb_sync_enabled() ? kmb_glr_check_error() : rc;
}

int kmb_glr_fwd(const KmbGLR *a) { return run(a, 0); }
int kmb_glr_bwd(const KmbGLR *a) { return run(a, 1); }

int kmb_glr_step(const KmbGLRStep *a) {
    KmbStage st;
    KmbGLR g; /* the checks of KmbGLR on the rows */
    const long lim = 1L << 31;
    int rc;
    if (!a) return kmb_fail(KMB_EINVAL, "glr: NULL arguments");
    if (a->rows < 0 || a->n_states < 0 || a->D <= 0)
        return kmb_fail(KMB_EINVAL, "glr: sizes must be positive");
    if (a->rows >= lim || a->n_states >= lim || a->D >= lim)
        return kmb_fail(KMB_EUNSUPPORTED, "glr: sizes too large");
    if (!a->slots && a->n_states < a->rows)
        return kmb_fail(KMB_EINVAL, "glr: fewer states than rows");
    if (a->rows && !a->state) return kmb_fail(KMB_EINVAL, "glr: state is required");
    if (misaligned(a->state, 4)) return kmb_fail(KMB_EINVAL, "glr: an fp32 tensor is not 4-byte aligned");
    if (misaligned(a->slots, 8)) return kmb_fail(KMB_EINVAL, "glr: slots are not 8-byte aligned");
    if (a->ld_state < a->D) return kmb_fail(KMB_EINVAL, "glr: state stride smaller than the state");
    memset(&g, 0, sizeof g);
    g.x = a->x;
    g.gate_r = a->gate_r;
    g.gate_i = a->gate_i;
    g.y = a->y;
    g.decay = a->decay;
    g.batch = 1;
    g.L = a->rows;
    g.D = a->D;
    g.scale = a->scale;
    g.type = a->type;
    if ((rc = validate(&g, 0))) return rc;
    const void *ptrs[] = {a->x.data, a->gate_r.data, a->gate_i.data, a->y.data,
                          a->decay,  a->state,       a->slots};
    if ((rc = kmb_check_device_ptrs("glr", ptrs, sizeof ptrs / sizeof *ptrs))) return rc;
    if ((rc = kmb_check_capture("glr", kmb_stream(), 0))) return rc;
    kmb_stage_begin(&st);
    rc = a->rows ? kmb_launch_glr_step(a, st.s) : KMB_OK;
    return kmb_stage_finish(&st, rc);
}
