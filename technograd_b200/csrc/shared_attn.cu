// shared_attn.cu -- tg_cuda_shared_attn: checks, how a call is cut, and its launches.
#include <algorithm>

#include "shared_attn.cuh"

namespace tgc {

extern template int shared_type<float>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);
extern template int shared_type<__half>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);
extern template int shared_type<__nv_bfloat16>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);

static int shared_check(const char *who, const tg_cuda_kv *c, const tg_cuda_prefix *x)
{
	if (!x) return set_err(TG_CUDA_EINVAL, "%s: NULL prefixes", who);
	if (x->groups < 0 || x->groups > c->seqs || x->max_shared < 0 || x->max_shared > c->max_len || x->max_own < 0 || x->always & ~1)
		return set_err(TG_CUDA_EINVAL, "%s: %d groups of %d sequences, at most %d positions shared and %d not, of %d (always %d)", who, x->groups, c->seqs, x->max_shared, x->max_own,
			       c->max_len, x->always);
	if (x->groups && (!x->first || !x->members || !x->shared || !x->group)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer in the prefixes", who);
	if (((uintptr_t)x->first | (uintptr_t)x->members | (uintptr_t)x->shared | (uintptr_t)x->group) & 3)
		return set_err(TG_CUDA_EINVAL, "%s: a pointer of the prefixes is not on a 4-byte boundary", who);
	return TG_CUDA_OK;
}

// What the sequences have of their own is often short, and a 128-row tile's chain is long: up to 64 rows take two 32-row tiles instead where
// there are few tiles in all. The whole call, us, 32-row against 128-row tiles (8 key heads of 128 dimensions, 42 rows, bf16, a prefix of 1024):
// 30.5 and 32.9 at 0.9 tiles an SM, 43.5 and 45.6 at 2.2, 65.7 and 78.2 at 4.3, 83.8 and 87.4 at 11, 157 and 188 at 13.8 (units of two
// tiles), but 67.6 and 60 at 14.3 (units of 33), 108 and 98 at 19, 190 and 182 at 21. 128 rows: 53.5 and 50 at 2.2.
constexpr int SHARED_MMA_ROWS = 64, SHARED_MMA_TILES = 14;

// Whether tree attention itself does it: nothing is shared, or reading a prefix for each sequence takes less time than two passes and
// their join. What each takes, from the bytes of keys and values it reads (as if all sequences had the longest prefix): tree
// attention 1 us for 8.5 MB (many of them from L2, since the sequences' tables name the same pages); here 5 us more to begin with, 1 for 4.5 MB, 20 ns
// a unit of a sequence and key head, and for f32 33 ns for each million operations of split products. Measured, us, here and tree attention
// (8 key heads of 128 dimensions, two query heads each, 65 positions of their own; bf16 unless f32): 4 sequences below 1024 positions 18.9 and
// 15.6, below 4096 19.9 and 19.6; 8 below 1024 19.1 and 16.7, below 2048 18.9 and 20.2; 16 below 512 18.5 and 16.8, below 1024 18.7 and 22.0; 64 below 256 30.6 and
// 28.0, below 1024 35.5 and 51.1; 64 in 32 groups below 2048 68 and 62, below 4096 95 and 107; f32: 4 below 4096 30 and 30, 16 below 1024 44 and 31,
// below 2048 47 and 55, 64 below 512 56 and 73. Over 370 other shapes (2 to 256 sequences of 1 to 64 tokens, 1 to 8 key heads and query heads each, 64 to 256
// dimensions, prefixes of 128 to 32768) it is 2.9% slower than the better of both each time, where always and never sharing are 18%. It is most wrong where
// it knows too little: many rows a sequence, whose tiles are full without sharing (190 of 32 tokens and 8 query heads a key head behind 696, pages of 24, 484
// here and 242 with tree attention, sharing chosen); 256 dimensions of 16 bits, whose prefixes are read for every 16 rows (13 of 4 tokens behind 10368 57 and
// 38, sharing chosen); f32 of many rows, whose products tree attention has too (213 of 8 query heads a key head behind 6240 238 and 426, tree attention chosen).
static bool shared_tree(const tg_cuda_kv *c, const PgDrafts &d, const tg_cuda_prefix *x)
{
	if (!c->seqs || !x->groups || !x->max_shared) return true;
	if (x->always) return false;
	const double row = 2.0 * c->nkv * c->head_dim * pg_size(c->type), own = (double)c->seqs * std::min(x->max_own, c->max_len) * row;
	const double all = own + (double)c->seqs * x->max_shared * row, once = own + (double)x->groups * x->max_shared * row;
	const double products = c->type == TG_CUDA_F32 ? 4.0 * c->seqs * d.tokens * d.nq * c->head_dim * x->max_shared : 0;
	return all / 8.5e6 < 5 + once / 4.5e6 + 0.02 * c->seqs * c->nkv + products * 33e-9; // us
}

// The two passes follow one another, each on all SMs, or run next to each other, the prefixes on some SMs and the own positions on the rest
// (their CTAs do not fit on one SM, and the second pass's begin wherever the first's are not): then the shorter one's beginning, 8 us or more
// of looking things up, fetching and a first chain of products, costs nothing. What each is reckoned to take, in us of an SM: 2 a
// prefix's tile; of own positions 0.77 a tile of 16 rows by 64 keys, 1.2 of 32 rows, 1.5 of 128 rows by 128 keys, a unit's beginning counting as 3
// tiles or 6, and lengths as half of their bound. The constants are those that chose best over 119 shapes whose times differ (8 to 256
// sequences, 1 to 24 tokens, prefixes of 1024 to 16384, up to 1024 own positions): 1.8% slower than the better of both each time, where always next
// to each other is 2.5% and always one after the other 13.7%. E.g. (us, next to each other and one after the other) 64 sequences of up
// to 513 positions behind 2048 shared ones 35 and 45, with 16 SMs for the prefix (40 with 8, 46 with 64); 8 of 200 behind 131008 71 and 87, with 140;
// 256 of up to 1024 in 6 groups of up to 8000 176 and 158; 256 of 64 in 8 groups behind 16384 100 and 76.
static void shared_split(AttnPlan &pre, AttnPlan &own, int own_len)
{
	const double tiles = 0.5 * own_len / (own.tc ? 128 : 64); // (own_len is a bound)
	const double wo = own.units * (own.tc ? (tiles + 6) * 1.5 : (tiles + 3) * (own.mt == 1 ? 0.77 : 1.2)), wp = pre.units * 2.0;
	auto next_to = [&](int n) { return std::max(9 + wp / n, 8 + wo / (pre.sms - n)); };
	int n = 1;
	while (n + 1 < pre.sms && next_to(n + 1) <= next_to(n)) n++;
	if (next_to(n) >= 0.9 * (17 + (wp + wo) / pre.sms) || n >= pre.grid) return;
	const int rest = (pre.sms - n) * (own.wave / own.sms);
	pre.grid = n;
	if (own.units > rest) own.whole = 0, own.grid = rest;
	else if (own.grid > rest) own.grid = rest;
}

// What beginning a prefix's unit counts, in tiles of 128 rows: little where a CTA has few tiles and more shares shorten the call, more where shares
// would else be uneven. The whole call, us, with 2 and with 6 (8 key heads of 128 dimensions, two query heads each, bf16): 4 sequences below 4096 21.4 and
// 24.0, 8 below 2048 18.8 and 23.6, 16 below 8192 26.2 and 28.0, all below 7 tiles an SM; above, 8 below 16384 31.4 and 30.9, 8 of 8 query heads each below
// 65536 52.9 and 50.9, 40 of 21 tokens below 16384 193 and 191.
constexpr int SHARED_BEGIN = 2, SHARED_BEGIN_LONG = 6, SHARED_LONG = 7;

static int shared_plan(const char *who, const tg_cuda_kv *c, const PgDrafts &d, const tg_cuda_prefix *x, SharedPlan *o)
{
	tg_cuda_kv tail = *c;
	tail.max_len = std::min(c->max_len, x->max_own);
	int rc = attn_plan(who, &tail, d, &o->own);
	if (rc) return rc;
	if (o->own.tc && d.tokens * d.group <= SHARED_MMA_ROWS && (long long)o->own.units * ((tail.max_len + 127) / 128 + 1) <= (long long)SHARED_MMA_TILES * o->own.sms &&
	    (rc = attn_plan(who, &tail, d, &o->own, false)))
		return rc;
	AttnPlan &p = o->pre;
	p = {};
	p.dev = o->own.dev, p.sms = o->own.sms, o->dp = p.dp = o->own.dp;
	const long long rows = (long long)c->seqs * d.tokens * d.group, each = (rows + x->groups - 1) / x->groups; // each: an average group's (members are not the host's to know)
	p.tc = c->type != TG_CUDA_F32 && p.dp <= 128;
	p.mt = each <= 16 || p.dp == 256 ? 1 : 2;
	p.fma = c->type == TG_CUDA_F32 && each <= 8 ? each <= 4 ? 4 : 8 : 0;
	const int rt = p.tc ? 128 : p.fma ? p.fma : 16 * p.mt, tk = p.tc ? 128 : c->type == TG_CUDA_F32 ? 32 : 64;
	const long long pitch = rows / rt + x->groups + 1, units = c->nkv * pitch, tiles = ((long long)x->max_shared + tk - 1) / tk;
	if (units > 0x7fffffff || rows * c->nkv > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of %d tokens and %d heads", who, c->seqs, d.tokens, d.nq);
	p.least = 128 / tk, p.begin = p.tc && units * tiles > (long long)SHARED_LONG * p.sms ? SHARED_BEGIN_LONG : SHARED_BEGIN;
	p.slot = (size_t)(rt * p.dp + 2 * rt) * 4;
	const long long shares = (units * (tiles + p.begin) + p.least + p.begin - 1) / (p.least + p.begin), wave = (long long)p.sms * (p.tc || p.dp == 256 ? 1 : p.fma || (p.mt == 1 && c->type != TG_CUDA_F32) ? 3 : 2);
	p.grid = (int)std::min(shares, wave), p.units = (int)units, p.row_tiles = 1;
	if (p.tc) {
		AttnPlan reckoned = p;
		reckoned.units = (int)std::min<long long>(tiles * std::max((rows + rt - 1) / rt, (long long)x->groups) * c->nkv, 0x7fffffff); // tiles of all units
		shared_split(reckoned, o->own, tail.max_len);
		p.grid = reckoned.grid;
	}
	o->least_units = std::max((rows + rt - 1) / rt, (long long)x->groups) * c->nkv, o->pitch = (int)pitch, o->rows = rows * c->nkv;
	size_t at = 0;
	auto take = [&](size_t n) { const size_t was = at; at = (at + n + 255) / 256 * 256; return was; };
	for (int i = 0; i < 2; i++) {
		const AttnPlan &q = i ? o->own : o->pre;
		o->tab[i] = take((size_t)q.units * sizeof(int2)), o->whole_o[i] = take((size_t)o->rows * o->dp * 4), o->whole_ml[i] = take((size_t)o->rows * 8);
		o->part[i] = take(q.whole ? 0 : (size_t)q.grid * 2 * q.slot);
	}
	o->bytes = at;
	return TG_CUDA_OK;
}

} // namespace tgc

using namespace tgc;

extern "C" long long tg_cuda_shared_attn_workspace(const tg_cuda_kv *c, const tg_cuda_drafts *d, const tg_cuda_prefix *x)
{
	const char *who = "tg_cuda_shared_attn_workspace";
	clear_err();
	PgCache pc;
	PgDrafts pd;
	SharedPlan pl;
	int rc;
	if ((rc = pg_cache(who, c, &pc)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &pd)) || (rc = shared_check(who, c, x))) return rc;
	if (shared_tree(c, pd, x)) return tg_cuda_tree_attn_workspace(c, d);
	if ((rc = shared_plan(who, c, pd, x, &pl))) return rc;
	return (long long)pl.bytes;
}

extern "C" int tg_cuda_shared_attn(const tg_cuda_kv *c, const tg_cuda_drafts *d, const tg_cuda_prefix *x, void *out, long long out_seq,
				   long long out_tok, long long out_head, float *lse, void *work, long long work_bytes, void *stream)
{
	const char *who = "tg_cuda_shared_attn";
	clear_err();
	JoinArgs j = {};
	SharedArgs &p = j.own;
	SharedPlan pl;
	int rc, sms;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &p.d)) || (rc = shared_check(who, c, x))) return rc;
	if (shared_tree(c, p.d, x)) return tg_cuda_tree_attn(c, d, out, out_seq, out_tok, out_head, lse, work, work_bytes, stream);
	const int e = pg_size(c->type);
	if (!out || !lse) return set_err(TG_CUDA_EINVAL, "%s: NULL output", who);
	if (c->seqs <= 1) out_seq = 0; // strides along one element are not used
	if (d->tokens <= 1) out_tok = 0;
	if (d->nq <= 1) out_head = 0;
	if ((uintptr_t)lse & 3) return set_err(TG_CUDA_EINVAL, "%s: lse is not on a 4-byte boundary", who);
	if (((uintptr_t)out & 15) || ((out_seq | out_tok | out_head) * e & 15))
		return set_err(TG_CUDA_EINVAL, "%s: out rows must start on 16-byte boundaries", who);
	if ((rc = pg_apart(who, "out", c->head_dim, {out_seq, out_tok, out_head}, {c->seqs, d->tokens, d->nq}))) return rc;
	if ((rc = pg_device(who, &sms, &p.c.status)) || (rc = shared_plan(who, c, p.d, x, &pl))) return rc;
	if (!work || work_bytes < (long long)pl.bytes || ((uintptr_t)work & 15))
		return set_err(TG_CUDA_EINVAL, "%s: needs %zu bytes of 16-byte aligned scratch", who, pl.bytes);
	p.out = (char *)out, p.out_seq = out_seq * e, p.out_tok = out_tok * e, p.out_head = out_head * e, p.lse = lse, p.seqs = c->seqs;
	p.first = x->first, p.members = x->members, p.shared = x->shared, p.group = x->group, p.groups = x->groups, p.max_shared = x->max_shared;
	p.pitch = pl.pitch, p.align = 1;
	CUtensorMap maps[2] = {};
	PgBox box = {};
	const bool f16 = c->type == TG_CUDA_F16;
	if ((pl.pre.tc || pl.own.tc) && pg_map(&maps[0], p.c, p.c.k, f16, 64, &box) && pg_map(&maps[1], p.c, p.c.v, f16, 64, &box)) p.box = box, p.align = box.rows;
	j.pre = p;
	char *w = (char *)work;
	for (int i = 0; i < 2; i++) {
		const AttnPlan &q = i ? pl.own : pl.pre;
		SharedArgs &a = i ? j.own : j.pre;
		a.row_tiles = q.row_tiles, a.whole = q.whole, a.least = q.least, a.begin = q.begin, a.ctas = q.grid;
		a.tab = (int2 *)(w + pl.tab[i]), a.whole_o = (float *)(w + pl.whole_o[i]), a.whole_ml = (float2 *)(w + pl.whole_ml[i]), a.part = (float *)(w + pl.part[i]);
	}
	auto rt = [](const AttnPlan &q) { return q.tc ? 128 : q.fma ? q.fma : 16 * q.mt; };
	j.pre_rt = rt(pl.pre), j.own_rt = rt(pl.own), j.pre_ctas = pl.pre.grid, j.own_ctas = pl.own.grid, j.rows = pl.rows;
	cudaStream_t st = (cudaStream_t)stream;
	return c->type == TG_CUDA_F32 ? shared_type<float>(j, pl, maps, st) : f16 ? shared_type<__half>(j, pl, maps, st) : shared_type<__nv_bfloat16>(j, pl, maps, st);
}
