// tree_attn.cu -- tg_cuda_tree_attn: checks, how a call is cut, and its launch.
#include "tree_attn.cuh"

namespace tgc {

extern template int attn_type<float>(const AttnArgs &, const AttnPlan &, cudaStream_t);
extern template int attn_type<__half>(const AttnArgs &, const AttnPlan &, cudaStream_t);
extern template int attn_type<__nv_bfloat16>(const AttnArgs &, const AttnPlan &, cudaStream_t);

// A unit of at most so many keys is one CTA's: smaller shares would cost more in set-up and joining.
constexpr int ATTN_WHOLE = 256;
// 16-bit caches take the 128-row tiles of tree_attn_tc.cuh for more than 32 query rows per key head, which 32-row tiles read the
// cache twice for (34 rows: 8 sequences of up to 1280 positions 27.6 us against 33, 16 of up to 4001 65 against 123, 131009 positions
// 115 against 225); and for 17 to 32 rows where a CTA has more than ATTN_LONG tiles (32 rows, us, 128-row against 32-row
// tiles, 8 key heads of 128 dimensions, bf16: 27.3 and 27.1 at 5 tiles, 54.2 and 50.2 at 16, 62.5 and 63.7 at 19; 65.2 and 80.5 at 28,
// 80 and 110 at 42, 115 and 126 at 55, 211 and 259 at 125; at 64 dimensions 36.8 and 32.9 at 16, 48.4 and 51.4 at 28, 150 and 172 at
// 125). 16 rows are one 16-row tile, at 28 tiles a CTA 48 us against 65.
constexpr int ATTN_TC_ROWS = 32, ATTN_TC_ROWS_LONG = 16, ATTN_LONG = 24;

// What beginning a unit costs, in tiles. The 128-row tiles' is about 6 (their chain of products and the output), but
// where shares are short every CTA has such a start of its own and counting it only makes them uneven. 64 rows, us at 2, 4, 6 and
// 8: 27.5, 29.4, 31.5, 33.8 at 5 tiles a CTA (8 sequences of up to 1280 positions); 44.1, 40.6, 40.9, 40.5 at 10; 65, 65, 66.7, 70 at
// 19; 96, 78.7, 80.8, 84 at 42; 212, 206, 200, 200 at 125.
constexpr int ATTN_BEGIN = 2, ATTN_TC_BEGIN = 6, ATTN_TC_SHORT = 7;

int attn_plan(const char *who, const tg_cuda_kv *c, const PgDrafts &d, AttnPlan *o, bool wide)
{
	int rc = pg_sms(who, &o->dev, &o->sms);
	if (rc) return rc;
	const int rows = d.tokens * d.group;
	o->dp = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
	const long long tiles128 = (long long)c->seqs * c->nkv * ((c->max_len + 127) / 128 + 1); // the 128-row tiles, where one has all rows
	o->tc = wide && c->type != TG_CUDA_F32 && o->dp <= 128 && rows > (tiles128 > (long long)ATTN_LONG * o->sms ? ATTN_TC_ROWS_LONG : ATTN_TC_ROWS);
	o->mt = rows <= 16 || o->dp == 256 ? 1 : 2; // 256 dimensions of 32 rows do not fit in registers
	o->fma = c->type == TG_CUDA_F32 && rows <= 8 ? rows <= 4 ? 4 : 8 : 0;
	const int rt = o->tc ? 128 : o->fma ? o->fma : 16 * o->mt, tk = o->tc ? 128 : c->type == TG_CUDA_F32 ? 32 : 64;
	o->row_tiles = (rows + rt - 1) / rt;
	const long long units = (long long)c->seqs * c->nkv * o->row_tiles;
	const long long tiles = (c->max_len + tk - 1) / tk + (d.tokens + tk - 1) / tk;
	if (units > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of %d tokens and %d heads", who, c->seqs, d.tokens, d.nq);
	o->whole = tiles * tk <= ATTN_WHOLE, o->least = 128 / tk, o->begin = o->tc && units * tiles > (long long)ATTN_TC_SHORT * o->sms ? ATTN_TC_BEGIN : ATTN_BEGIN;
	o->slot = (size_t)(rt * o->dp + 2 * rt) * 4;
	const long long shares = (units * (tiles + o->begin) + o->least + o->begin - 1) / (o->least + o->begin), wave = (long long)o->sms * (o->tc || o->dp == 256 ? 1 : o->fma || (o->mt == 1 && c->type != TG_CUDA_F32) ? 3 : 2); // the tiles' CTAS
	o->grid = (int)(o->whole ? units : shares < wave ? shares : wave);
	o->wave = (int)wave, o->units = (int)units, o->by_unit = !o->whole && units <= o->grid;
	return TG_CUDA_OK;
}

} // namespace tgc

using namespace tgc;

extern "C" long long tg_cuda_tree_attn_workspace(const tg_cuda_kv *c, const tg_cuda_drafts *d)
{
	const char *who = "tg_cuda_tree_attn_workspace";
	clear_err();
	PgCache pc;
	PgDrafts pd;
	AttnPlan pl;
	int rc;
	if ((rc = pg_cache(who, c, &pc)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &pd))) return rc;
	if (c->seqs == 0) return 0;
	if ((rc = attn_plan(who, c, pd, &pl))) return rc;
	return (long long)pl.bytes();
}

extern "C" int tg_cuda_tree_attn(const tg_cuda_kv *c, const tg_cuda_drafts *d, void *out, long long out_seq, long long out_tok,
				 long long out_head, float *lse, void *work, long long work_bytes, void *stream)
{
	const char *who = "tg_cuda_tree_attn";
	clear_err();
	AttnArgs p = {};
	AttnPlan pl;
	int rc, sms;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &p.d))) return rc;
	const int e = pg_size(c->type);
	if (c->seqs && (!out || !lse)) return set_err(TG_CUDA_EINVAL, "%s: NULL output", who);
	if (c->seqs <= 1) out_seq = 0; // strides along one element are not used
	if (d->tokens <= 1) out_tok = 0;
	if (d->nq <= 1) out_head = 0;
	if ((uintptr_t)lse & 3) return set_err(TG_CUDA_EINVAL, "%s: lse is not on a 4-byte boundary", who);
	if (((uintptr_t)out & 15) || ((out_seq | out_tok | out_head) * e & 15))
		return set_err(TG_CUDA_EINVAL, "%s: out rows must start on 16-byte boundaries", who);
	if ((rc = pg_apart(who, "out", c->head_dim, {out_seq, out_tok, out_head}, {c->seqs, d->tokens, d->nq}))) return rc;
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0 || (rc = attn_plan(who, c, p.d, &pl))) return rc;
	const size_t need = pl.bytes();
	if (need && (!work || work_bytes < (long long)need || ((uintptr_t)work & 15)))
		return set_err(TG_CUDA_EINVAL, "%s: needs %zu bytes of 16-byte aligned scratch", who, need);
	p.out = (char *)out, p.out_seq = out_seq * e, p.out_tok = out_tok * e, p.out_head = out_head * e, p.lse = lse;
	p.seqs = c->seqs, p.row_tiles = pl.row_tiles, p.whole = pl.whole, p.least = pl.least, p.begin = pl.begin, p.by_unit = pl.by_unit, p.ctas = pl.grid;
	p.split = (int4 *)work, p.part = (float *)((char *)work + (size_t)pl.grid * sizeof(int4));
	cudaStream_t st = (cudaStream_t)stream;
	return c->type == TG_CUDA_F32 ? attn_type<float>(p, pl, st) : c->type == TG_CUDA_F16 ? attn_type<__half>(p, pl, st) : attn_type<__nv_bfloat16>(p, pl, st);
}
