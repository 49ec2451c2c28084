// rope.cu -- rotary positions: tg_cuda_rope, and tg_cuda_kv_append, which writes new tokens' keys and values into a
// paged cache with the norm and the rotation on the way.
#include <algorithm>

#include "paged.cuh"

namespace tgc {

// Rows that the kernel moves: heads of every token, from src to dst and, with `cache`, to the token's cache row.
struct TurnRows {
	const char *src;
	char *dst, *pool;                  // either may be NULL
	long long s_seq, s_tok, s_head, d_seq, d_tok, d_head; // bytes
	const float *norm;                 // [dim] or NULL
	int heads, turn;
};

struct TurnArgs {
	PgCache c;                         // table and len NULL: no cache
	TurnRows rows[3];
	int nrows, heads;                  // of them, and all their heads
	const double *freq;
	const int *pos;
	long long pos_seq;
	const int *count;
	int *len_out;
	long long all;                     // seqs * tokens
	int tokens, dim, part, inverse, per; // per: tokens of a block
	float gain, eps;
};

// cos and sin of pos * freq. The angle is taken in turns, as 64 bits behind the point: whole turns fall off the product by
// themselves, so a far position's angle is as exact as a near one's (2^-55 turns of the frequency times the position).
// What is left of the nearest quarter turn has 24 significant bits of its own in f32.
__device__ __forceinline__ float2 turn_of(double freq, int pos)
{
	double x = freq * 0.15915494309189535; // 1 / 2 pi
	x -= rint(x);
	const unsigned long long f = (unsigned long long)__double2ll_rn(x * 0x1p63) << 1;
	const unsigned long long t = f * (unsigned long long)(long long)pos;
	const unsigned q = (unsigned)((t + (1ull << 61)) >> 62);
	float s, c;
	sincospif((float)(long long)(t - ((unsigned long long)q << 62)) * 0x1p-63f, &s, &c);
	const float a = q & 1 ? s : c, b = q & 1 ? c : s;
	return make_float2(q == 1 || q == 2 ? -a : a, q & 2 ? -b : b);
}

enum { TURN_HALF, TURN_PAIRS, TURN_ANY }; // halves that begin at 16-byte pieces; neighbours; halves that begin anywhere

struct TurnToken {
	long long b, row; // its sequence, and its cache row in bytes (-1: none)
	int i, live;
};

// A thread has two 16-byte pieces of a row (TURN_HALF: the two that turn with each other), a row's threads lie in one
// warp, so that a row may be written where it is read. cos and sin of a token are computed once for all its heads.
template <class T, int FORM, bool NORM>
__global__ void __launch_bounds__(256) k_turn(const TurnArgs p, int lanes, int lg)
{
	constexpr int E = 16 / (int)sizeof(T);
	extern __shared__ __align__(16) float2 cs[]; // [per][n * E]
	__shared__ TurnToken tok[8];
	const int tid = threadIdx.x, half = p.part >> 1, n = (half + E - 1) / E, nch = p.dim / E, width = FORM == TURN_ANY ? half : n * E;
	const long long t0 = (long long)blockIdx.x * p.per;
	const int per = (int)min((long long)p.per, p.all - t0);
	if (tid < per) {
		TurnToken k;
		k.b = (t0 + tid) / p.tokens, k.i = (int)(t0 + tid - k.b * p.tokens), k.live = 1, k.row = -1;
		if (p.count) k.live = k.i < p.count[k.b];
		if (p.c.len) {
			const int len = p.c.length((int)k.b), all = p.count ? max(0, min(p.count[k.b], p.tokens)) : p.tokens;
			const long long at = (long long)len + k.i;
			if (k.i == 0) p.len_out[k.b] = len + all;
			if (k.live) {
				if (at >= (long long)p.c.page * p.c.cols || at > 0x7fffffff) p.c.report(PG_ROOM);
				else k.row = p.c.row(p.c.table + k.b * p.c.cols, (int)at);
			}
		}
		tok[tid] = k;
	}
	for (int x = tid; x < per * width; x += 256) {
		const int t = per == 1 ? 0 : x / width, a = x - t * width;
		const long long b = (t0 + t) / p.tokens;
		const int i = (int)(t0 + t - b * p.tokens);
		float2 v = make_float2(1, 0);
		if (a < half) {
			const int at = p.pos ? p.pos[b * p.pos_seq + i] : p.c.len ? (int)((unsigned)p.c.length((int)b) + (unsigned)i) : i;
			v = turn_of(p.freq[a], at);
			v.x *= p.gain, v.y *= p.inverse ? -p.gain : p.gain;
		}
		// the pairs of a thread in 16-byte pieces, the pieces of neighbouring threads next to each other
		cs[t * width + (FORM == TURN_ANY ? a : (((a % E) >> 1) * n + a / E) * 2 + (a & 1))] = v;
	}
	__syncthreads();
	const int mine = tid & (lanes - 1), total = per * p.heads;
	for (int r0 = 0; r0 < total; r0 += 256 >> lg) {
		const int r = r0 + (tid >> lg), t = min(r, total - 1) / p.heads;
		int h = min(r, total - 1) - t * p.heads, g = 0;
		while (g + 1 < p.nrows && h >= p.rows[g].heads) h -= p.rows[g++].heads;
		const TurnRows &w = p.rows[g];
		const TurnToken k = tok[t];
		const bool turn = w.turn && FORM != TURN_ANY && mine < n;
		const int c0 = FORM != TURN_HALF ? 2 * mine : mine < n ? mine : 2 * mine, c1 = FORM == TURN_HALF && mine < n ? mine + n : c0 + 1;
		const bool in = r < total, h0 = in && c0 < nch, h1 = in && c1 < nch;
		const char *src = w.src + k.b * w.s_seq + k.i * w.s_tok + h * w.s_head;
		uint4 raw[2] = {};
		if (k.live && h0) raw[0] = *(const uint4 *)(src + c0 * 16);
		if (k.live && h1) raw[1] = *(const uint4 *)(src + c1 * 16);
		float x[2 * E];
#pragma unroll
		for (int e = 0; e < 2 * E; e++) x[e] = PgElem<T>::get(((const T *)raw)[e]);
		float inv = 1;
		if constexpr (NORM) {
			float ss = 0;
#pragma unroll
			for (int e = 0; e < 2 * E; e++) ss = fmaf(x[e], x[e], ss);
			for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
			if (w.norm) {
				inv = __frsqrt_rn(ss / (float)p.dim + p.eps);
#pragma unroll
				for (int e = 0; e < 2 * E; e++) {
					const int c = e < E ? c0 : c1;
					x[e] = x[e] * inv * (c < nch ? w.norm[c * E + e % E] : 0);
				}
			}
		}
		if constexpr (FORM == TURN_ANY) {
			if (w.turn && k.live) {
#pragma unroll
				for (int e = 0; e < 2 * E; e++) {
					const int el = (e < E ? c0 : c1) * E + e % E, a = el < half ? el : el - half, other = el < half ? el + half : a;
					if (in && el < p.part) {
						float y = PgElem<T>::get(((const T *)src)[other]);
						if (NORM && w.norm) y = y * inv * w.norm[other];
						const float2 v = cs[t * width + a];
						x[e] = fmaf(x[e], v.x, el < half ? -(y * v.y) : y * v.y);
					}
				}
			}
		} else if (turn) {
			const float4 *table = (const float4 *)(cs + t * width) + mine;
#pragma unroll
			for (int i = 0; i < E / 2; i++) {
				const float4 v = table[i * n];
				const int a0 = FORM == TURN_HALF ? 2 * i : 4 * i, b0 = FORM == TURN_HALF ? a0 + E : a0 + 1, a1 = FORM == TURN_HALF ? a0 + 1 : a0 + 2, b1 = FORM == TURN_HALF ? b0 + 1 : a0 + 3;
				const float p0 = x[a0], q0 = x[b0], p1 = x[a1], q1 = x[b1];
				x[a0] = fmaf(p0, v.x, -(q0 * v.y)), x[b0] = fmaf(p0, v.y, q0 * v.x);
				x[a1] = fmaf(p1, v.z, -(q1 * v.w)), x[b1] = fmaf(p1, v.w, q1 * v.z);
			}
		}
		if (w.turn || (NORM && w.norm)) { // (else the bits pass as they are)
#pragma unroll
			for (int e = 0; e < 2 * E; e++) ((T *)raw)[e] = PgElem<T>::put(x[e]);
		}
		__syncwarp(); // the row has been read
		if (w.dst) {
			char *to = w.dst + k.b * w.d_seq + k.i * w.d_tok + h * w.d_head;
			if (h0) *(uint4 *)(to + c0 * 16) = k.live ? raw[0] : make_uint4(0, 0, 0, 0);
			if (h1) *(uint4 *)(to + c1 * 16) = k.live ? raw[1] : make_uint4(0, 0, 0, 0);
		}
		if (w.pool && k.row >= 0) {
			char *to = w.pool + k.row + h * p.c.head_b;
			if (h0) *(uint4 *)(to + c0 * 16) = raw[0];
			if (h1) *(uint4 *)(to + c1 * 16) = raw[1];
		}
	}
}

static int turn_check(const char *who, const tg_cuda_rotary *r, int head_dim, int e, int seqs, int tokens, TurnArgs *p)
{
	if (r->dim < 0 || r->dim > head_dim || r->dim & 1) return set_err(TG_CUDA_EINVAL, "%s: %d elements of a head of %d turn", who, r->dim, head_dim);
	if (r->interleaved & ~1 || r->inverse & ~1) return set_err(TG_CUDA_EINVAL, "%s: interleaved %d, inverse %d", who, r->interleaved, r->inverse);
	if (r->dim && !r->freq) return set_err(TG_CUDA_EINVAL, "%s: NULL frequencies", who);
	if (((uintptr_t)r->freq & 7) || ((uintptr_t)r->pos & 3)) return set_err(TG_CUDA_EINVAL, "%s: freq (8 bytes) or pos (4) is not on a boundary of its type", who);
	if (r->pos && seqs > 1 && r->pos_seq < 0) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	p->part = r->dim, p->inverse = r->inverse, p->gain = r->gain, p->freq = r->freq, p->pos = r->pos, p->pos_seq = seqs > 1 ? r->pos_seq : 0;
	return TG_CUDA_OK;
}

template <class T, int FORM>
static int turn_launch(TurnArgs &p, bool norm, cudaStream_t st)
{
	constexpr int E = 16 / (int)sizeof(T);
	const int items = (p.dim / E + 1) / 2;
	int lg = 0;
	while (1 << lg < items) lg++;
	p.heads = 0;
	for (int g = 0; g < p.nrows; g++) p.heads += p.rows[g].heads;
	p.per = std::max(1, std::min(8, 256 / std::max(1, std::min(256, p.heads << lg))));
	const long long blocks = (p.all + p.per - 1) / p.per;
	if (blocks > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "rotary positions: %lld tokens", p.all);
	const int width = FORM == TURN_ANY ? p.part / 2 : (p.part / 2 + E - 1) / E * E;
	const size_t smem = (size_t)p.per * width * sizeof(float2);
	if (norm) k_turn<T, FORM, true><<<(unsigned)blocks, 256, smem, st>>>(p, 1 << lg, lg);
	else k_turn<T, FORM, false><<<(unsigned)blocks, 256, smem, st>>>(p, 1 << lg, lg);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

template <class T> static int turn_form(TurnArgs &p, int pairs, bool norm, cudaStream_t st)
{
	if (pairs) return turn_launch<T, TURN_PAIRS>(p, norm, st);
	return p.part * (int)sizeof(T) % 32 ? turn_launch<T, TURN_ANY>(p, norm, st) : turn_launch<T, TURN_HALF>(p, norm, st);
}

static int turn_type(TurnArgs &p, int type, int pairs, bool norm, void *stream)
{
	cudaStream_t st = (cudaStream_t)stream;
	return type == TG_CUDA_F32 ? turn_form<float>(p, pairs, norm, st) : type == TG_CUDA_F16 ? turn_form<__half>(p, pairs, norm, st) : turn_form<__nv_bfloat16>(p, pairs, norm, st);
}

// An output's rows: on 16-byte boundaries, and none over another. Strides along one element are not used.
static int turn_out(const char *who, const char *what, void *out, long long (&s)[3], int seqs, int tokens, int heads, int dim, int e)
{
	const int n[3] = { seqs, tokens, heads };
	for (int i = 0; i < 3; i++)
		if (n[i] <= 1) s[i] = 0;
	if (((uintptr_t)out & 15) || ((s[0] | s[1] | s[2]) * e & 15)) return set_err(TG_CUDA_EINVAL, "%s: %s rows must start on 16-byte boundaries", who, what);
	return pg_apart(who, what, dim, { s[0], s[1], s[2] }, { seqs, tokens, heads });
}

} // namespace tgc

using namespace tgc;

extern "C" int tg_cuda_rope(const tg_cuda_rotary *r, int type, int seqs, int tokens, int heads, int head_dim, const void *x, long long x_seq,
			    long long x_tok, long long x_head, void *out, long long out_seq, long long out_tok, long long out_head, void *stream)
{
	const char *who = "tg_cuda_rope";
	clear_err();
	if (!r) return set_err(TG_CUDA_EINVAL, "%s: NULL rotation", who);
	if (type != TG_CUDA_F32 && type != TG_CUDA_F16 && type != TG_CUDA_BF16) return set_err(TG_CUDA_EINVAL, "%s: element type %d", who, type);
	const int e = pg_size(type);
	if (seqs < 0 || tokens < 0 || heads < 0 || heads > 1 << 20) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of %d tokens and %d heads", who, seqs, tokens, heads);
	if (head_dim <= 0 || head_dim > 256 || head_dim * e % 16) return set_err(TG_CUDA_EINVAL, "%s: head_dim %d: at most 256, in rows of a multiple of 16 bytes", who, head_dim);
	TurnArgs p = {};
	int rc, dev, sms;
	if ((rc = turn_check(who, r, head_dim, e, seqs, tokens, &p))) return rc;
	const bool none = !seqs || !tokens || !heads;
	if (!none && (!x || !out)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	long long s[3] = { seqs > 1 ? x_seq : 0, tokens > 1 ? x_tok : 0, heads > 1 ? x_head : 0 }, o[3] = { out_seq, out_tok, out_head };
	if (s[0] < 0 || s[1] < 0 || s[2] < 0) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	if (((uintptr_t)x & 15) || ((s[0] | s[1] | s[2]) * e & 15)) return set_err(TG_CUDA_EINVAL, "%s: x rows must start on 16-byte boundaries", who);
	if (!none && (rc = turn_out(who, "out", out, o, seqs, tokens, heads, head_dim, e))) return rc;
	if ((rc = pg_sms(who, &dev, &sms)) || none) return rc;
	p.rows[0] = { (const char *)x, (char *)out, nullptr, s[0] * e, s[1] * e, s[2] * e, o[0] * e, o[1] * e, o[2] * e, nullptr, heads, 1 };
	p.nrows = 1, p.all = (long long)seqs * tokens, p.tokens = tokens, p.dim = head_dim;
	return turn_type(p, type, r->interleaved, false, stream);
}

extern "C" int tg_cuda_kv_append(const tg_cuda_kv *c, const tg_cuda_drafts *d, const tg_cuda_rotary *r, const float *q_norm, const float *k_norm,
				 float eps, void *q_out, long long q_out_seq, long long q_out_tok, long long q_out_head, void *k_out,
				 long long k_out_seq, long long k_out_tok, long long k_out_head, int *len_out, void *stream)
{
	const char *who = "tg_cuda_kv_append";
	clear_err();
	TurnArgs p = {};
	PgDrafts pd;
	int rc, sms;
	const bool q = d && d->q;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_K | PG_USE_V | (q ? PG_USE_Q : 0), 0, &pd))) return rc;
	const int e = pg_size(c->type);
	if (c->nkv > 1 << 20) return set_err(TG_CUDA_EINVAL, "%s: nkv %d is over 2^20", who, c->nkv);
	p.gain = 1;
	if (r && (rc = turn_check(who, r, c->head_dim, e, c->seqs, d->tokens, &p))) return rc;
	if (c->seqs && (!len_out || !d->q != !q_out)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (len_out == c->len && c->seqs) return set_err(TG_CUDA_EINVAL, "%s: len_out may not be the cache's len", who);
	if (((uintptr_t)len_out | (uintptr_t)q_norm | (uintptr_t)k_norm) & 3) return set_err(TG_CUDA_EINVAL, "%s: a pointer is not on a 4-byte boundary", who);
	if (q_norm && !q) return set_err(TG_CUDA_EINVAL, "%s: q_norm without q", who);
	long long qo[3] = { q_out_seq, q_out_tok, q_out_head }, ko[3] = { k_out_seq, k_out_tok, k_out_head };
	if (q && (rc = turn_out(who, "q_out", q_out, qo, c->seqs, d->tokens, d->nq, c->head_dim, e))) return rc;
	if (k_out && (rc = turn_out(who, "k_out", k_out, ko, c->seqs, d->tokens, c->nkv, c->head_dim, e))) return rc;
	if ((rc = pg_apart(who, "the cache", c->head_dim, {c->page_stride, c->head_stride, c->pos_stride}, {c->pages, c->nkv, c->page}))) return rc;
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0) return rc;
	if (q) p.rows[p.nrows++] = { pd.q, (char *)q_out, nullptr, pd.q_seq, pd.q_tok, pd.q_head, qo[0] * e, qo[1] * e, qo[2] * e, q_norm, d->nq, r && r->dim };
	p.rows[p.nrows++] = { pd.k, (char *)k_out, p.c.k, pd.kv_seq, pd.kv_tok, pd.kv_head, ko[0] * e, ko[1] * e, ko[2] * e, k_norm, c->nkv, r && r->dim };
	p.rows[p.nrows++] = { pd.v, nullptr, p.c.v, pd.kv_seq, pd.kv_tok, pd.kv_head, 0, 0, 0, nullptr, c->nkv, 0 };
	p.count = d->count, p.len_out = len_out, p.all = (long long)c->seqs * d->tokens, p.tokens = d->tokens, p.dim = c->head_dim, p.eps = eps;
	return turn_type(p, c->type, r && r->interleaved, q_norm || k_norm, stream);
}
