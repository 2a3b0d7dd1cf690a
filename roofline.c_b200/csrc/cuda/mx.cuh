// mx.cuh -- what the microscaled operators (mx.cu, mx_linear.cu) share.
#pragma once

#include "lm.cuh"
#include "mx_index.h"

namespace tcg {

// Checks of a held matrix that need no device.
inline bool mx_check(const char *who, const char *name, const tcg_mx_t *m)
{
    if (!m) return fail("%s: no %s", who, name);
    if (m->bits != 4 && m->bits != 8) return fail("%s: %s in %d bits: 4 or 8", who, name, m->bits);
    if (m->rows < 0 || m->rows > TCG_MX_MAX_ROWS || m->cols < 1 || m->cols > TCG_MX_MAX_COLS)
        return fail("%s: %s of %d rows and %d columns", who, name, m->rows, m->cols);
    if (m->rows && (!m->codes || !m->scales)) return fail("%s: %s has no codes or no scales", who, name);
    if ((uintptr_t)m->codes % 32 || (uintptr_t)m->scales % 16)
        return fail("%s: %s needs codes on a 32-byte and scales on a 16-byte boundary", who, name);
    return true;
}

// A plain matrix's pointer and stride against its type, rows and columns.
inline bool mx_rows(const char *who, const char *name, const void *p, int rows, int64_t cols, int64_t ld, ggml_type_t t)
{
    if (!rows) return true;
    if (!p) return fail("%s: no %s", who, name);
    if ((uintptr_t)p % lm_type_size(t)) return fail("%s: misaligned %s", who, name);
    if (ld < cols && rows > 1)
        return fail("%s: %s rows of %lld columns do not fit a stride of %lld", who, name, (long long)cols, (long long)ld);
    return true;
}

}  // namespace tcg
