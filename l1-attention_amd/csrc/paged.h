// The paged 8-bit cache as the kernels see it: l1attn_cache of the C header with 32-bit sizes, passed by value.
#pragma once
#include "common.h"
#include "../../include/l1attn_hip.h"

struct L1Cache {
	int N, P, Hk, W, Wv, pk, pv, rows, M;  // pages, tokens of a page, heads, widths, bytes of a row (a multiple of 16), table rows, pages of a row
	int8_t *k, *v;
	float *ks, *vs;
	int32_t *table, *lens, *refs, *free, *n_free;
};

static inline int l1_cache_args(const l1attn_cache* c, L1Cache* a)
{
	if (!c) return L1ATTN_ERR_ARG;
	if (c->n_pages < 0 || c->Hk < 1 || c->W < 1 || c->Wv < 1 || c->rows < 0 || c->row_pages < 0) return L1ATTN_ERR_ARG;
	if (c->page != 16 && c->page != 32 && c->page != 64) return L1ATTN_ERR_ARG;
	if (c->W > 128 || c->Wv > 128 || c->Hk > 1024 || c->n_pages > (1 << 28) || c->rows > (1 << 24) || c->row_pages > (1 << 24)) return L1ATTN_ERR_RANGE;
	if (c->row_pages * c->page > (1 << 30)) return L1ATTN_ERR_RANGE;
	if (c->n_pages && (!c->k_pages || !c->v_pages || !c->k_scale || !c->v_scale || !c->refs || !c->free_pages)) return L1ATTN_ERR_ARG;
	if (!c->n_free || (c->rows && (!c->lens || (c->row_pages && !c->table)))) return L1ATTN_ERR_ARG;
	if (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15) return L1ATTN_ERR_ARG;
	a->N = (int)c->n_pages; a->P = (int)c->page; a->Hk = (int)c->Hk; a->W = (int)c->W; a->Wv = (int)c->Wv;
	a->pk = (int)l1_align_up((size_t)c->W, 16); a->pv = (int)l1_align_up((size_t)c->Wv, 16);
	a->rows = (int)c->rows; a->M = (int)c->row_pages;
	a->k = c->k_pages; a->v = c->v_pages; a->ks = c->k_scale; a->vs = c->v_scale;
	a->table = c->table; a->lens = c->lens; a->refs = c->refs; a->free = c->free_pages; a->n_free = c->n_free;
	return L1ATTN_OK;
}
