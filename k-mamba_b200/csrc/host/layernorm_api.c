/*
 * Layer norm entry points (kmamba_b200.h): argument checks, the workspace,
 * and the launch.  No counterpart in the reference, whose blocks have no
 * norm.
 */
#include <math.h>
#include <stdint.h>

#include "../kmb_internal.h"

static size_t elem(int type) { return type == KMB_BF16 ? 2 : 4; }
static int known(int type) { return type == KMB_F32 || type == KMB_BF16; }
static int misaligned(const void *p, size_t n) { return p && ((uintptr_t)p & (n - 1)) != 0; }

size_t kmb_layernorm_workspace_bytes(const KmbLayerNorm *a) {
    if (!a || a->rows < 0 || a->D <= 0 || a->rows >= (1L << 31) || a->D >= (1L << 31)) return 0;
    return kmb_layernorm_scratch_bytes(a->rows, a->D);
}

static int validate(const KmbLayerNorm *a, int bwd) {
    if (!a) return kmb_fail(KMB_EINVAL, "layernorm: NULL arguments");
    if (a->rows < 0 || a->D <= 0) return kmb_fail(KMB_EINVAL, "layernorm: sizes must be positive");
    if (a->rows >= (1L << 31) || a->D >= (1L << 31))
        return kmb_fail(KMB_EUNSUPPORTED, "layernorm: rows and D must be below 2^31");
    if (!known(a->x_type) || !known(a->y_type))
        return kmb_fail(KMB_EINVAL, "layernorm: unknown element type");
    if (!(a->eps >= 0.f) || isinf(a->eps))
        return kmb_fail(KMB_EINVAL, "layernorm: eps must be finite and not negative");
    if (a->accumulate != 0 && a->accumulate != 1)
        return kmb_fail(KMB_EINVAL, "layernorm: accumulate must be 0 or 1");
    if (a->rows) {
        if (!a->x) return kmb_fail(KMB_EINVAL, "layernorm: x is required");
        if (!bwd && !a->y) return kmb_fail(KMB_EINVAL, "layernorm: y is required");
        if (bwd && (!a->dy || !a->dx)) return kmb_fail(KMB_EINVAL, "layernorm: dy and dx are required");
    }
    if (bwd && !a->mean != !a->rstd)
        return kmb_fail(KMB_EINVAL, "layernorm: mean and rstd must be given together");
    if (a->ld_x < a->D || (!bwd && a->ld_y < a->D) ||
        (bwd && (a->ld_dy < a->D || a->ld_dx < a->D || (a->dres && a->ld_dres < a->D))))
        return kmb_fail(KMB_EINVAL, "layernorm: row stride smaller than the row");
    const size_t xs = elem(a->x_type), ys = elem(a->y_type);
    if (misaligned(a->x, xs) || misaligned(a->weight, 4) || misaligned(a->mean, 4) ||
        misaligned(a->rstd, 4) || (!bwd && (misaligned(a->y, ys) || misaligned(a->bias, 4))) ||
        (bwd && (misaligned(a->dy, ys) || misaligned(a->dx, xs) || misaligned(a->dres, xs) ||
                 misaligned(a->dweight, 4) || misaligned(a->dbias, 4))))
        return kmb_fail(KMB_EINVAL, "layernorm: a tensor is not aligned to its element");
    /* an output over an input has its type and stride */
    const int same = a->x_type == a->y_type;
    if (a->rows && ((!bwd && a->y == a->x && !(same && a->ld_y == a->ld_x)) ||
                    (bwd && ((a->dx == a->x && a->ld_dx != a->ld_x) ||
                             (a->dx == a->dy && !(same && a->ld_dx == a->ld_dy)) ||
                             (a->dx == a->dres && a->ld_dx != a->ld_dres)))))
        return kmb_fail(KMB_EINVAL, "layernorm: an output over an input of another type or stride");
    return KMB_OK;
}

int kmb_layernorm_fwd(const KmbLayerNorm *a) {
    KmbStage st;
    int rc = validate(a, 0);
    if (rc) return rc;
    const void *ptrs[] = {a->x, a->weight, a->bias, a->y, a->mean, a->rstd};
    if ((rc = kmb_check_device_ptrs("layernorm", ptrs, sizeof ptrs / sizeof *ptrs))) return rc;
    if ((rc = kmb_check_capture("layernorm", kmb_stream(), 0))) return rc;
    kmb_stage_begin(&st);
    rc = a->rows ? kmb_launch_layernorm_fwd(a, st.s) : KMB_OK;
    rc = kmb_stage_finish(&st, rc);
    return !rc && kmb_sync_enabled() ? kmb_layernorm_check_error() : rc;
}

int kmb_layernorm_bwd(const KmbLayerNorm *a) {
    KmbStage st;
    KmbLayerNorm d;
    int rc = validate(a, 1);
    if (rc) return rc;
    const int sums = a->dweight || a->dbias;
    const size_t need = sums ? kmb_layernorm_workspace_bytes(a) : 0;
    if (need && a->workspace) {
        if (a->workspace_bytes < need)
            return kmb_fail(KMB_EINVAL, "layernorm: workspace of %zu bytes, %zu needed",
                            a->workspace_bytes, need);
        if (misaligned(a->workspace, 16))
            return kmb_fail(KMB_EINVAL, "layernorm: workspace must be 16-byte aligned");
    }
    const void *ptrs[] = {a->x,  a->weight,  a->mean,  a->rstd, a->dy, a->dres,
                          a->dx, a->dweight, a->dbias, need ? a->workspace : NULL};
    if ((rc = kmb_check_device_ptrs("layernorm", ptrs, sizeof ptrs / sizeof *ptrs))) return rc;
    if ((rc = kmb_check_capture("layernorm", kmb_stream(), need && !a->workspace))) return rc;
    kmb_stage_begin(&st);
    d = *a;
    if (need && !d.workspace) d.workspace = kmb_scratch(&st, need);
    rc = st.status ? st.status : kmb_launch_layernorm_bwd(&d, st.s);
    rc = kmb_stage_finish(&st, rc);
    return !rc && kmb_sync_enabled() ? kmb_layernorm_check_error() : rc;
}
