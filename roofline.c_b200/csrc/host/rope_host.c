/* rope_host.c -- rotary positions: the host plan (tcg_rope_t).
 *
 * A plan holds, for each rotated pair, the revolutions it makes per position:
 * turns[i] = base^(-2i / n_rot) / (2 pi), changed by the context-extension
 * rules. Revolutions rather than radians, because the kernel then reduces an
 * angle exactly: frac(p * turns[i]) in 64 bits, with no division by 2 pi at
 * far positions. Host only, no GPU; the struct is copied into each launch.
 *
 * The context rules work on the turns a pair makes over the trained context,
 * orig_ctx * turns[i], which is what their published forms (wavelength
 * against context length) say in other words. */
#include "tcg.h"
#include "tcg_internal.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

static const double TWO_PI = 6.283185307179586476925286766559;

static bool plan_ok(const tcg_rope_t *r, const char *who)
{
    if (!r) return host_fail("%s: no plan", who);
    if (r->n_rot < 2 || r->n_rot > TCG_ROPE_MAX_DIM || (r->n_rot & 1))
        return host_fail("%s: the plan is not initialised", who);
    return true;
}

static bool factor_ok(double f, const char *who)
{
    if (!(f > 0.0) || !isfinite(f)) return host_fail("%s: factor %g is not a positive number", who, f);
    return true;
}

bool tcg_rope_init(tcg_rope_t *r, int head_dim, int n_rot, int layout, double base)
{
    if (!r) return host_fail("tcg_rope_init: no plan");
    if (head_dim < 2 || head_dim > TCG_ROPE_MAX_DIM || (head_dim & 1))
        return host_fail("tcg_rope_init: head_dim %d is not an even number in 2 .. %d", head_dim, TCG_ROPE_MAX_DIM);
    if (n_rot < 2 || n_rot > head_dim || (n_rot & 1))
        return host_fail("tcg_rope_init: n_rot %d is not an even number in 2 .. %d", n_rot, head_dim);
    if (layout != TCG_ROPE_INTERLEAVED && layout != TCG_ROPE_HALF)
        return host_fail("tcg_rope_init: unknown pair layout %d", layout);
    if (!(base > 0.0) || !isfinite(base)) return host_fail("tcg_rope_init: base %g is not a positive number", base);
    memset(r, 0, sizeof *r);
    r->head_dim = head_dim;
    r->n_rot = n_rot;
    r->layout = layout;
    r->mscale = 1.0f;
    r->base = base;
    for (int i = 0; i < n_rot / 2; i++) r->turns[i] = pow(base, -2.0 * i / n_rot) / TWO_PI;
    return true;
}

bool tcg_rope_scale_linear(tcg_rope_t *r, double factor)
{
    if (!plan_ok(r, "tcg_rope_scale_linear") || !factor_ok(factor, "tcg_rope_scale_linear")) return false;
    for (int i = 0; i < r->n_rot / 2; i++) r->turns[i] /= factor;
    return true;
}

/* The pair index (a real number) at which a pair of the unscaled base makes
 * `n` turns over ctx tokens: ctx * base^(-2i / n_rot) / (2 pi) = n. */
static double pair_of_turns(const tcg_rope_t *r, double n, double ctx)
{
    return r->n_rot * log(ctx / (n * TWO_PI)) / (2.0 * log(r->base));
}

bool tcg_rope_scale_yarn(tcg_rope_t *r, double factor, int orig_ctx, double beta_fast, double beta_slow,
                         double attn_factor)
{
    const char *who = "tcg_rope_scale_yarn";
    if (!plan_ok(r, who) || !factor_ok(factor, who)) return false;
    if (orig_ctx < 1) return host_fail("%s: original context %d is not positive", who, orig_ctx);
    if (!(beta_slow > 0.0) || !(beta_fast >= beta_slow) || !isfinite(beta_fast))
        return host_fail("%s: needs 0 < beta_slow <= beta_fast, got %g and %g", who, beta_slow, beta_fast);
    if (!(attn_factor >= 0.0) || !isfinite(attn_factor))
        return host_fail("%s: attn_factor %g is negative or not finite", who, attn_factor);
    if (r->base <= 1.0) return host_fail("%s: needs a base above 1, got %g", who, r->base);
    const double low = fmax(0.0, floor(pair_of_turns(r, beta_fast, orig_ctx)));
    const double high = fmin(r->n_rot - 1.0, ceil(pair_of_turns(r, beta_slow, orig_ctx)));
    const double width = fmax(high - low, 0.001);
    for (int i = 0; i < r->n_rot / 2; i++) {
        const double slow = fmin(fmax((i - low) / width, 0.0), 1.0);
        r->turns[i] *= (1.0 - slow) + slow / factor;
    }
    r->mscale *= (float)(attn_factor > 0.0 ? attn_factor : factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0);
    return true;
}

bool tcg_rope_scale_bands(tcg_rope_t *r, double factor, int orig_ctx, double low, double high)
{
    const char *who = "tcg_rope_scale_bands";
    if (!plan_ok(r, who) || !factor_ok(factor, who)) return false;
    if (orig_ctx < 1) return host_fail("%s: original context %d is not positive", who, orig_ctx);
    if (!(low >= 0.0) || !(high > low) || !isfinite(high))
        return host_fail("%s: needs 0 <= low < high, got %g and %g", who, low, high);
    for (int i = 0; i < r->n_rot / 2; i++) {
        const double keep = fmin(fmax((orig_ctx * r->turns[i] - low) / (high - low), 0.0), 1.0);
        r->turns[i] *= keep + (1.0 - keep) / factor;
    }
    return true;
}

bool tcg_rope_scale_factors(tcg_rope_t *r, const float *f, int n)
{
    const char *who = "tcg_rope_scale_factors";
    if (!plan_ok(r, who)) return false;
    if (!f || n != r->n_rot / 2) return host_fail("%s: %d factors for %d pairs", who, f ? n : 0, r->n_rot / 2);
    for (int i = 0; i < n; i++)
        if (!(f[i] > 0.0f) || !isfinite(f[i])) return host_fail("%s: factor %d is %g", who, i, (double)f[i]);
    for (int i = 0; i < n; i++) r->turns[i] /= f[i];
    return true;
}

/* A number of the metadata, of any scalar type; `fallback` when the key is absent, false when it holds something else. */
static bool number(const gguf_t *g, const char *key, double fallback, double *out)
{
    const gguf_kv_t *kv = gguf_find(g, key);
    int64_t i;
    float f;
    *out = fallback;
    if (!kv) return true;
    if (kv->type == GGUF_T_FLOAT64) *out = kv->v.f64;
    else if (gguf_get_f32(g, key, &f)) *out = (double)f;
    else if (kv->type != GGUF_T_BOOL && gguf_get_i64(g, key, &i)) *out = (double)i;
    else return false;
    return true;
}

/* What else a file says of positions must not be passed over, since it changes the angles or the magnitude: every key
 * under <arch>.rope. is one that the plan follows, says nothing (the value beside it), or is refused, and so is every
 * tensor of rotary factors but rope_freqs.weight. False names the first one that is refused. */
static bool all_known(const gguf_t *g, const char *arch, const char *who)
{
    static const char *const followed[] = { "dimension_count", "freq_base", "scaling.type", "scaling.factor",
                                            "scaling.original_context_length", "scaling.attn_factor",
                                            "scaling.finetuned" };       /* of the weights: it changes no angle */
    static const struct { const char *name; double neutral; } idle[] = {
        { "scale_linear", 1.0 }, { "scaling.yarn_ext_factor", 1.0 }, { "scaling.yarn_attn_factor", 1.0 },
        { "scaling.yarn_beta_fast", 32.0 }, { "scaling.yarn_beta_slow", 1.0 }, { "scaling.yarn_log_multiplier", 0.0 } };
    char start[80];
    const size_t skip = (size_t)snprintf(start, sizeof start, "%s.rope.", arch);
    for (uint64_t i = 0; i < g->n_kv; i++) {
        const gguf_str_t key = g->kv[i].key;
        if (!key.ptr || key.len < skip || memcmp(key.ptr, start, skip)) continue;
        const gguf_str_t name = { key.ptr + skip, key.len - skip };
        bool known = false;
        for (size_t j = 0; j < sizeof followed / sizeof *followed; j++) known = known || gguf_str_eq(name, followed[j]);
        for (size_t j = 0; j < sizeof idle / sizeof *idle; j++) {
            char full[160];
            double v;
            snprintf(full, sizeof full, "%s%s", start, idle[j].name);
            known = known || (gguf_str_eq(name, idle[j].name) && number(g, full, 0.0, &v) && v == idle[j].neutral);
        }
        if (!known) return host_fail("%s: '%.*s' is not followed here (tcg_rope_init and tcg_rope_scale_* take any rule)", who,
                                     (int)(key.len < 100 ? key.len : 100), key.ptr);
    }
    for (uint64_t i = 0; i < g->n_tensors; i++) {
        const gguf_str_t name = g->tensors[i].name;
        if (!name.ptr || gguf_str_eq(name, "rope_freqs.weight")) continue;
        for (uint64_t at = 0; at + 5 <= name.len; at++)
            if (!memcmp(name.ptr + at, "rope_", 5))
                return host_fail("%s: the tensor '%.*s' is not followed here", who, (int)(name.len < 100 ? name.len : 100),
                                 name.ptr);
    }
    return true;
}

bool tcg_rope_from_gguf(tcg_rope_t *r, const gguf_t *g, int layout)
{
    const char *who = "tcg_rope_from_gguf";
    if (!r || !g) return host_fail("%s: no plan or no file", who);
    gguf_str_t a;
    char arch[64], key[128];
    if (!gguf_get_str(g, "general.architecture", &a) || a.len == 0 || a.len >= sizeof arch)
        return host_fail("%s: no general.architecture", who);
    memcpy(arch, a.ptr, a.len);
    arch[a.len] = '\0';
#define KEY(name) (snprintf(key, sizeof key, "%s." name, arch), key)
    const uint64_t heads = gguf_u64_or(g, KEY("attention.head_count"), 0), wide = gguf_u64_or(g, KEY("embedding_length"), 0);
    uint64_t d = gguf_u64_or(g, KEY("attention.key_length"), heads && wide % heads == 0 ? wide / heads : 0);
    if (d == 0) return host_fail("%s: %s has no attention.key_length, nor an embedding_length and head_count that give it", who, arch);
    const uint64_t n_rot = gguf_u64_or(g, KEY("rope.dimension_count"), d);
    if (d > TCG_ROPE_MAX_DIM || n_rot > d) return host_fail("%s: head length %llu, %llu of it rotated", who,
                                                                 (unsigned long long)d, (unsigned long long)n_rot);
    if (!all_known(g, arch, who)) return false;
    double base, factor, attn;
    if (!number(g, KEY("rope.freq_base"), 10000.0, &base) || !number(g, KEY("rope.scaling.factor"), 0.0, &factor) ||
        !number(g, KEY("rope.scaling.attn_factor"), 1.0, &attn))
        return host_fail("%s: %s is not a number", who, key);
    tcg_rope_t plan;                            /* *r changes only when everything is read */
    if (!tcg_rope_init(&plan, (int)d, (int)n_rot, layout, base)) return false;
    const gguf_tensor_t *t = gguf_tensor(g, "rope_freqs.weight");
    if (t) {
        if (t->type != GGML_TYPE_F32 || !t->data || t->n_elem != n_rot / 2)
            return host_fail("%s: rope_freqs.weight is not %llu F32 values", who, (unsigned long long)(n_rot / 2));
        float f[TCG_ROPE_MAX_DIM / 2];
        memcpy(f, t->data, (size_t)t->n_elem * sizeof(float));
        if (!tcg_rope_scale_factors(&plan, f, (int)t->n_elem)) return false;
    }
    gguf_str_t kind = { NULL, 0 };
    if (gguf_find(g, KEY("rope.scaling.type")) && !gguf_get_str(g, key, &kind)) return host_fail("%s: %s is not a text", who, key);
    const bool yarn = gguf_str_eq(kind, "yarn");
    if (!yarn && attn != 1.0) return host_fail("%s: attn_factor %g without a rope.scaling.type of yarn", who, attn);
    if (!kind.ptr) {
        /* some readers take a factor without a type as linear, some as none */
        if (factor != 0.0 && factor != 1.0) return host_fail("%s: a rope.scaling.factor of %g without a type", who, factor);
    } else if (!gguf_str_eq(kind, "none")) {
        if (gguf_str_eq(kind, "linear")) {
            if (!tcg_rope_scale_linear(&plan, factor)) return false;
        } else if (yarn) {
            const uint64_t ctx = gguf_u64_or(g, KEY("rope.scaling.original_context_length"),
                                             gguf_u64_or(g, KEY("context_length"), 0));
            if (ctx > 0x7fffffffu) return host_fail("%s: original context %llu", who, (unsigned long long)ctx);
            /* a positive attn_factor scales the rule's own 0.1 ln(factor) + 1 */
            if (!(attn > 0.0)) return host_fail("%s: attn_factor %g", who, attn);
            if (!tcg_rope_scale_yarn(&plan, factor, (int)ctx, 32.0, 1.0, 0.0)) return false;
            plan.mscale *= (float)attn;
        } else {
            return host_fail("%s: unknown rope.scaling.type '%.*s'", who, (int)(kind.len < 32 ? kind.len : 32), kind.ptr);
        }
    }
#undef KEY
    *r = plan;
    return true;
}
