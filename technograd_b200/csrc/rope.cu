// rope.cu -- rotary positions: tg_cuda_rope, and tg_cuda_kv_append, which writes new tokens' keys and values into a
// paged cache with the norm and the rotation on the way.
#include <algorithm>

#include "mma_sync.cuh"
#include "paged.cuh"

namespace tgc {

// Rows that the kernel moves: heads of every token, from src to dst and, keys and values, to the token's cache row in pool.
struct TurnRows {
	const char *src;
	char *dst, *pool;                  // dst NULL: not wanted
	long long s_seq, s_tok, s_head, d_seq, d_tok, d_head; // bytes
	const float *norm;                 // [dim] or NULL
	int heads, turn, cached;           // cached: into the pool
	int aligned, chunks;               // norm lies on a 16-byte boundary; warps that have a token's rows of this kind
};

struct TurnArgs {
	PgCache c;                         // table and len NULL: no cache
	TurnRows rows[3];
	int nrows;
	int chunks;                        // warps that have a token's rows
	const double *freq;
	const int *pos;
	long long pos_seq;
	const int *count;
	int *len_out;
	long long all;                     // seqs * tokens
	int tokens, dim, part, inverse;
	float gain, eps, over_dim;         // 1 / dim
};

// cos and sin of pos * freq. The angle is taken in turns, as 64 bits behind the point: whole turns fall off the product by
// themselves, so a far position's angle is as exact as a near one's. freq / 2 pi is taken in two parts, of twice 53 bits, and rounded to
// 2^-65 turns, which a position of 32 bits makes 2^-33; the product's first 32 bits are rounded to 2^-33 too: 2^-29.3 radians
// together (for frequencies below 2^40; one part and no rounding left 2^-22 at positions of 2^31). Bits behind the point come from sums with
// a number whose last bit is theirs: conversions between f64 and integers, at a quarter of f64's rate, took 99 us where these take 87 (k_turn_any's
// example, below; 83 with one part).
// These 32 bits are a quarter turn and a rest of at most an eighth, x = 2 pi rest, whose sine and cosine
// are their Taylor series up to x^9 and x^10: what is left out is below (pi/4)^11 / 11! = 1.8e-9 and (pi/4)^12 / 12! = 1.2e-10, and
// over all 2^30 rests they are off by 1.10e-7 and 1.02e-7 at most, below 2^-23.
__device__ __forceinline__ float2 turn_of(double freq, long long pos)
{
	constexpr double WHOLE = 0x1.8p52, UPPER = 0x1.8p20, LOWER = 0x1.8p-12; // last bits 1, 2^-32 and 2^-64
	const double turns = freq * 0.15915494309189535; // 1 / 2 pi; what it is short of that is the next line's factor
	const double low = fma(freq, -9.839338337591243e-18, fma(freq, 0.15915494309189535, -turns));
	const double f = turns - ((turns + WHOLE) - WHOLE);
	if (isnan(f)) return make_float2(NAN, NAN); // freq is an infinity or no number
	const double u0 = f + UPPER, u1 = (f - (u0 - UPPER)) + low + LOWER;
	const unsigned long long u = ((unsigned long long)__double_as_longlong(u0) << 32) + (unsigned long long)(__double_as_longlong(u1) - __double_as_longlong(LOWER));
	const unsigned t = (unsigned)((u * (unsigned long long)pos + (1ull << 31)) >> 32), q = (t + (1u << 29)) >> 30;
	const float x = (float)(int)(t - (q << 30)) * 1.4629180792671596e-9f, z = x * x; // 2 pi / 2^32
	const float s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1 / 362880.f, -1 / 5040.f), 1 / 120.f), -1 / 6.f), 1.f);
	const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1 / 3628800.f, 1 / 40320.f), -1 / 720.f), 1 / 24.f), -0.5f), 1.f);
	const float a = q & 1 ? s : c, b = q & 1 ? c : s;
	return make_float2((q + 1) & 2 ? -a : a, q & 2 ? -b : b);
}

// 16 bytes of elements as pairs of f32, and back, rounded to nearest
__device__ __forceinline__ void turn_get(float2 (&x)[2], const uint4 &w, float)
{
	x[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y)), x[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ void turn_get(float2 (&x)[4], const uint4 &w, __nv_bfloat16)
{
	const uint32_t v[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
	for (int i = 0; i < 4; i++) x[i] = make_float2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u));
}
__device__ __forceinline__ void turn_get(float2 (&x)[4], const uint4 &w, __half)
{
	const uint32_t v[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
	for (int i = 0; i < 4; i++) x[i] = __half22float2(*(const __half2 *)&v[i]);
}
__device__ __forceinline__ uint4 turn_put(const float2 (&x)[2], float)
{
	return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
}
template <class T> __device__ __forceinline__ uint4 turn_put(const float2 (&x)[4], T)
{
	return make_uint4(pack16(x[0].x, x[0].y, T()), pack16(x[1].x, x[1].y, T()), pack16(x[2].x, x[2].y, T()), pack16(x[3].x, x[3].y, T()));
}

enum { TURN_HALF, TURN_PAIRS }; // halves that begin at 16-byte pieces; neighbours
constexpr int TURN_ANY_ROWS = 4; // rows of a warp in k_turn_any

// A row's norm, its inverse: the sum over the `lanes` threads that have the row's elements x and y.
template <int N> __device__ __forceinline__ float turn_norm(const float2 (&x)[N], const float2 (&y)[N], int lanes, float over_dim, float eps)
{
	float2 s = make_float2(0, 0);
#pragma unroll
	for (int e = 0; e < N; e++) s = fma2(x[e], x[e], fma2(y[e], y[e], s));
	float ss = s.x + s.y;
#pragma unroll
	for (int o = 16; o; o >>= 1)
		if (o < lanes) ss += __shfl_xor_sync(~0u, ss, o);
	return rsqrtf(fmaf(ss, over_dim, eps));
}

// a / b of numbers that nearly always fit 32 bits (a 64-bit division is a long chain of instructions)
__device__ __forceinline__ long long over(long long a, int b) { return a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b); }

// Four weights of a norm, which may begin at any word
__device__ __forceinline__ float4 turn_weights(const TurnRows &w, int at)
{
	return w.aligned ? *(const float4 *)(w.norm + at) : make_float4(w.norm[at], w.norm[at + 1], w.norm[at + 2], w.norm[at + 3]);
}

// Position of a token: behind a long cache past 32 bits
__device__ __forceinline__ long long turn_pos(const TurnArgs &p, long long b, int i, int len)
{
	return p.pos ? p.pos[b * p.pos_seq + i] : (long long)len + i;
}

// A warp has UN rounds of one token's rows of one kind (q, k or v): 1 << lg threads a row, each with two 16-byte pieces, those
// that turn with each other. So a thread has the same E pairs in all its rows and keeps their cos and sin in registers; the warp's
// threads of one place compute PART of them each and pass them round. No shared memory, no barrier, and all rounds'
// loads on their way at once. A row's pieces are read and written by the same thread, reads first, so that a row may
// be written where it is read. FULL: every thread of a row has two pieces.
// What bounds it: HBM where there are many tokens, latency where there are few; with norms the instructions, about 700 a warp of four
// rounds. Measured (bf16, 128 dimensions): 8 x 6001 tokens of 16 heads 60 us, 6.5 TB/s (117 with cos and sin in shared memory and a
// barrier); 16 prompts of up to 2047 tokens, 16 query heads and 8 key heads normed and rotated into the cache, 111 us, 4.2 TB/s (118 with
// all of a token's rows in one warp, which then looks up each kind's strides as it goes).
template <class T, int FORM, bool NORM, int PART, int UN, bool FULL>
__global__ void __launch_bounds__(128, 5) k_turn(const TurnArgs p, int lg)
{
	constexpr int E = 16 / (int)sizeof(T);
	const int lane = threadIdx.x & 31, lanes = 1 << lg, mine = lane & (lanes - 1), at = lane >> lg, half = p.part >> 1, n = (half + E - 1) / E, nch = p.dim / E;
	const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), w = over(item, p.chunks);
	if (w >= p.all) return;
	int chunk = (int)(item - w * p.chunks), g = 0;
	const bool begin = chunk == 0;
	while (chunk >= p.rows[g].chunks) chunk -= p.rows[g++].chunks;
	const long long b = over(w, p.tokens);
	const int i = (int)(w - b * p.tokens), h0 = chunk * (UN << (5 - lg)) + at, heads = p.rows[g].heads, turns = p.rows[g].turn;
	const float *norm = NORM ? p.rows[g].norm : nullptr;
	const int c0 = FORM == TURN_PAIRS ? 2 * mine : mine < n ? mine : 2 * mine, c1 = FORM == TURN_HALF && mine < n ? mine + n : c0 + 1, apart = (c1 - c0) * 16;
	const bool have0 = FULL || c0 < nch, have1 = FULL || c1 < nch;
	int cnt = p.tokens, len = 0;
	if (p.count) cnt = max(0, min(p.count[b], p.tokens));
	const bool live = i < cnt;
	uint4 raw[UN][2];
	{
		const long long s_head = p.rows[g].s_head;
		const char *src = p.rows[g].src + b * p.rows[g].s_seq + i * p.rows[g].s_tok + h0 * s_head + c0 * 16;
#pragma unroll
		for (int u = 0; u < UN; u++) {
			const bool in = live && h0 + (u << (5 - lg)) < heads;
			if (!FULL || !live) raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
			if (in && have0) raw[u][0] = __ldcs((const uint4 *)src);
			if (in && have1) raw[u][1] = __ldcs((const uint4 *)(src + apart));
			src += s_head << (5 - lg);
		}
	}
	char *pool = nullptr;
	if (p.c.len) {
		len = p.c.length((int)b);
		if (begin && i == 0 && lane == 0) p.len_out[b] = p.c.grown(len, cnt);
		if (p.rows[g].cached && live) {
			const long long to = (long long)len + i;
			if (to >= (long long)p.c.page * p.c.cols || to > 0x7fffffff) p.c.report(PG_ROOM);
			else {
				const long long row = p.c.row(p.c.table + b * p.c.cols, (int)to);
				if (row >= 0) pool = p.rows[g].pool + row + h0 * p.c.head_b + c0 * 16;
			}
		}
	}
	if (live && (turns || norm)) { // (else the bits pass as they are)
		float2 c[E / 2], s[E / 2], ns[E / 2], wx[E / 2], wy[E / 2]; // two pairs' cos, sin and -sin; the pieces' weights
		if (turns) {
			const long long pos = turn_pos(p, b, i, len);
			float2 own[PART];
#pragma unroll
			for (int x = 0; x < PART; x++) {
				const int e = at * PART + x, a = mine * E + e;
				own[x] = make_float2(1, 0);
				if (e < E && a < half) {
					own[x] = turn_of(p.freq[a], pos);
					own[x].x *= p.gain, own[x].y *= p.inverse ? -p.gain : p.gain;
				}
			}
#pragma unroll
			for (int e = 0; e < E; e += 2) {
				const int from = (e / PART << lg) + mine, next = ((e + 1) / PART << lg) + mine;
				c[e / 2] = make_float2(__shfl_sync(~0u, own[e % PART].x, from), __shfl_sync(~0u, own[(e + 1) % PART].x, next));
				s[e / 2] = make_float2(__shfl_sync(~0u, own[e % PART].y, from), __shfl_sync(~0u, own[(e + 1) % PART].y, next));
				ns[e / 2] = make_float2(-s[e / 2].x, -s[e / 2].y);
			}
		}
		if (norm) {
#pragma unroll
			for (int e = 0; e < E / 2; e += 2) {
				const float4 v = have0 ? turn_weights(p.rows[g], c0 * E + 2 * e) : make_float4(0, 0, 0, 0), z = have1 ? turn_weights(p.rows[g], c1 * E + 2 * e) : make_float4(0, 0, 0, 0);
				wx[e] = make_float2(v.x, v.y), wx[e + 1] = make_float2(v.z, v.w);
				wy[e] = make_float2(z.x, z.y), wy[e + 1] = make_float2(z.z, z.w);
			}
		}
		const bool turn = turns && (FULL && FORM == TURN_HALF && 2 * n == nch || mine < n);
#pragma unroll
		for (int u = 0; u < UN; u++) {
			if (u && h0 - at + (u << (5 - lg)) >= heads) break; // the whole warp
			float2 x[E / 2], y[E / 2];
			turn_get(x, raw[u][0], T()), turn_get(y, raw[u][1], T());
			if (NORM && norm) {
				const float inv = turn_norm(x, y, lanes, p.over_dim, p.eps);
				const float2 two = make_float2(inv, inv);
#pragma unroll
				for (int e = 0; e < E / 2; e++) x[e] = mul2(mul2(x[e], two), wx[e]), y[e] = mul2(mul2(y[e], two), wy[e]);
			}
			if (turn) {
				if constexpr (FORM == TURN_HALF) {
#pragma unroll
					for (int e = 0; e < E / 2; e++) {
						const float2 v = x[e];
						x[e] = fma2(y[e], ns[e], mul2(v, c[e])), y[e] = fma2(v, s[e], mul2(y[e], c[e]));
					}
				} else {
#pragma unroll
					for (int e = 0; e < E; e++) {
						if (mine * E + e >= half) break; // what passes, infinities too
						float2 &v = e < E / 2 ? x[e] : y[e - E / 2];
						const float cc = e % 2 ? c[e / 2].y : c[e / 2].x, ss = e % 2 ? s[e / 2].y : s[e / 2].x;
						v = make_float2(fmaf(v.x, cc, -(v.y * ss)), fmaf(v.x, ss, v.y * cc));
					}
				}
			}
			raw[u][0] = turn_put(x, T()), raw[u][1] = turn_put(y, T());
		}
	}
	if (p.rows[g].dst) {
		const long long d_head = p.rows[g].d_head;
		char *dst = p.rows[g].dst + b * p.rows[g].d_seq + i * p.rows[g].d_tok + h0 * d_head + c0 * 16;
#pragma unroll
		for (int u = 0; u < UN; u++) {
			const bool in = h0 + (u << (5 - lg)) < heads;
			if (in && have0) *(uint4 *)dst = raw[u][0];
			if (in && have1) *(uint4 *)(dst + apart) = raw[u][1];
			dst += d_head << (5 - lg);
		}
	}
	if (pool) {
#pragma unroll
		for (int u = 0; u < UN; u++) {
			const bool in = h0 + (u << (5 - lg)) < heads;
			if (in && have0) *(uint4 *)pool = raw[u][0];
			if (in && have1) *(uint4 *)(pool + apart) = raw[u][1];
			pool += p.c.head_b << (5 - lg);
		}
	}
}

// Halves that begin within a 16-byte piece: a warp a row, element by element. A thread has the pairs lane, lane + 32, ... of a row
// (behind the rotated part, neighbours), and so the same in all rows of one kind that the warp has. NI: pairs of a thread.
// What bounds it: the instructions of 2-byte loads and stores. Measured: 16 x 2000 tokens of 16 heads of 128 dimensions, 100 of them
// rotated, bf16 87 us, f32 89 us (114 and 169 with whole pieces whose elements look their partners up one by one).
template <class T, bool NORM, int NI>
__global__ void __launch_bounds__(128) k_turn_any(const TurnArgs p)
{
	const int lane = threadIdx.x & 31, half = p.part >> 1, pairs = p.dim / 2;
	const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), w = over(item, p.chunks);
	if (w >= p.all) return;
	int chunk = (int)(item - w * p.chunks), g = 0;
	const bool begin = chunk == 0;
	while (chunk >= p.rows[g].chunks) chunk -= p.rows[g++].chunks;
	const TurnRows &k = p.rows[g];
	const long long b = over(w, p.tokens);
	const int i = (int)(w - b * p.tokens), first = chunk * TURN_ANY_ROWS, last = min(k.heads, first + TURN_ANY_ROWS);
	int cnt = p.tokens, len = 0;
	if (p.count) cnt = max(0, min(p.count[b], p.tokens));
	const bool live = i < cnt;
	long long row = -1;
	if (p.c.len) {
		len = p.c.length((int)b);
		if (begin && i == 0 && lane == 0) p.len_out[b] = p.c.grown(len, cnt);
		if (k.cached && live) {
			const long long to = (long long)len + i;
			if (to >= (long long)p.c.page * p.c.cols || to > 0x7fffffff) p.c.report(PG_ROOM);
			else row = p.c.row(p.c.table + b * p.c.cols, (int)to);
		}
	}
	int one[NI], two[NI]; // the elements of a pair, -1: none
	float2 cs[NI], norm[NI];
#pragma unroll
	for (int n = 0; n < NI; n++) {
		const int a = n * 32 + lane;
		one[n] = a >= pairs ? -1 : a < half ? a : 2 * a;
		two[n] = a < half ? a + half : 2 * a + 1;
		cs[n] = make_float2(1, 0), norm[n] = make_float2(1, 1);
		if (k.turn && live && a < half) {
			cs[n] = turn_of(p.freq[a], turn_pos(p, b, i, len));
			cs[n].x *= p.gain, cs[n].y *= p.inverse ? -p.gain : p.gain;
		}
		if (NORM && k.norm && one[n] >= 0) norm[n] = make_float2(k.norm[one[n]], k.norm[two[n]]);
	}
	const char *src = k.src + b * k.s_seq + i * k.s_tok;
	char *dst = k.dst + b * k.d_seq + i * k.d_tok, *pool = k.pool + row;
	T rows_x[TURN_ANY_ROWS][NI], rows_y[TURN_ANY_ROWS][NI]; // all on their way at once
#pragma unroll
	for (int r = 0; r < TURN_ANY_ROWS; r++) {
		const T *s = (const T *)(src + (first + r) * k.s_head);
#pragma unroll
		for (int n = 0; n < NI; n++) {
			rows_x[r][n] = rows_y[r][n] = PgElem<T>::put(0);
			if (live && first + r < last && one[n] >= 0) rows_x[r][n] = s[one[n]], rows_y[r][n] = s[two[n]];
		}
	}
#pragma unroll
	for (int r = 0; r < TURN_ANY_ROWS; r++) {
		const int h = first + r;
		if (h >= last) break;
		T(&x)[NI] = rows_x[r], (&y)[NI] = rows_y[r];
		if (live && (k.turn || (NORM && k.norm))) { // (else the bits pass as they are)
			float u[NI], v[NI], inv = 1;
#pragma unroll
			for (int n = 0; n < NI; n++) u[n] = PgElem<T>::get(x[n]), v[n] = PgElem<T>::get(y[n]);
			if (NORM && k.norm) {
				float ss = 0;
#pragma unroll
				for (int n = 0; n < NI; n++) ss = fmaf(u[n], u[n], fmaf(v[n], v[n], ss));
#pragma unroll
				for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
				inv = rsqrtf(fmaf(ss, p.over_dim, p.eps));
			}
#pragma unroll
			for (int n = 0; n < NI; n++) {
				if (NORM && k.norm) u[n] = u[n] * inv * norm[n].x, v[n] = v[n] * inv * norm[n].y;
				const float a = u[n], z = v[n];
				if (n * 32 + lane < half) u[n] = fmaf(a, cs[n].x, -(z * cs[n].y)), v[n] = fmaf(a, cs[n].y, z * cs[n].x); // (what passes does, infinities too)
				x[n] = PgElem<T>::put(u[n]), y[n] = PgElem<T>::put(v[n]);
			}
		}
		if (k.dst) {
			T *to = (T *)(dst + h * k.d_head);
#pragma unroll
			for (int n = 0; n < NI; n++)
				if (one[n] >= 0) to[one[n]] = x[n], to[two[n]] = y[n];
		}
		if (row >= 0) {
			T *to = (T *)(pool + h * p.c.head_b);
#pragma unroll
			for (int n = 0; n < NI; n++)
				if (one[n] >= 0) to[one[n]] = x[n], to[two[n]] = y[n];
		}
	}
}

static int turn_check(const char *who, const tg_cuda_rotary *r, int head_dim, int seqs, TurnArgs *p)
{
	if (r->dim < 0 || r->dim > head_dim || r->dim & 1) return set_err(TG_CUDA_EINVAL, "%s: %d elements of a head of %d turn", who, r->dim, head_dim);
	if (r->interleaved & ~1 || r->inverse & ~1) return set_err(TG_CUDA_EINVAL, "%s: interleaved %d, inverse %d", who, r->interleaved, r->inverse);
	if (r->dim && !r->freq) return set_err(TG_CUDA_EINVAL, "%s: NULL frequencies", who);
	if (((uintptr_t)r->freq & 7) || ((uintptr_t)r->pos & 3)) return set_err(TG_CUDA_EINVAL, "%s: freq (8 bytes) or pos (4) is not on a boundary of its type", who);
	if (r->pos && seqs > 1 && r->pos_seq < 0) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	p->part = r->dim, p->inverse = r->inverse, p->gain = r->gain, p->freq = r->freq, p->pos = r->pos, p->pos_seq = seqs > 1 ? r->pos_seq : 0;
	return TG_CUDA_OK;
}

// Whether a warp takes four rounds rather than two: where there are many bytes, and that saves a third of the warps, or with norms, whose weights
// are then looked up half as often, a quarter (else its places are mostly empty). Measured, us, two rounds and four (bf16, 128 dimensions, four rounds being 16
// rows): 16 heads of 4096 tokens 8.1 and 8.3, of 32768 43.8 and 42.0; 32 heads of 2048 8.1 and 8.4, of 32768 84.3 and 80.5; 8 heads of 32768 23.6 and
// 27.6, 1 head 18.3 and 22.9. Appends of 16 prompts of 2047 tokens with norms: 32 query heads over 8 191 and 161, 16 over 8 129 and 119, 8 key heads
// alone 64 and 68; without, 16 over 8 89 and 94, 32 over 4 120 and 117. f32, 16 over 8: 173 and 161 with norms, 160 and 161
// without; 2 prompts of 1024 13.1 and 12.3, 11.2 and 9.7 (bf16 10.0 and 10.9, 7.0 and 8.0).
constexpr long long TURN_MANY = 24 << 20; // bytes

static bool turn_four(const TurnArgs &p, bool norm, int lg, int e)
{
	const int r = 1 << (5 - lg); // rows of a round
	long long rows = 0, two = 0, four = 0; // of a token: rows, and the warps that have them
	for (int g = 0; g < p.nrows; g++) {
		const int h = p.rows[g].heads;
		rows += h, two += (h + 2 * r - 1) / (2 * r), four += (h + 4 * r - 1) / (4 * r);
	}
	return p.all >= TURN_MANY / (rows * p.dim * e) && (norm ? four * 4 <= two * 3 : four * 3 <= two * 2);
}

static int turn_grid(long long blocks)
{
	return blocks > 0x7fffffff ? set_err(TG_CUDA_EINVAL, "rotary positions: a grid of %lld blocks", blocks) : TG_CUDA_OK;
}

template <class T, int FORM, int PART, int UN, bool FULL>
static int turn_launch(TurnArgs &p, bool norm, int lg, cudaStream_t st)
{
	p.chunks = 0;
	for (int g = 0; g < p.nrows; g++) p.chunks += p.rows[g].chunks = (p.rows[g].heads + (UN << (5 - lg)) - 1) / (UN << (5 - lg));
	const __int128 items = (__int128)p.all * p.chunks;
	const long long blocks = items > 0x1ffffffffll ? 0x80000000ll : (long long)(items + 3) / 4;
	if (turn_grid(blocks)) return TG_CUDA_EINVAL;
	if (norm) k_turn<T, FORM, true, PART, UN, FULL><<<(unsigned)blocks, 128, 0, st>>>(p, lg);
	else k_turn<T, FORM, false, PART, UN, FULL><<<(unsigned)blocks, 128, 0, st>>>(p, lg);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

template <class T, int FORM, int PART>
static int turn_rounds(TurnArgs &p, bool norm, int lg, cudaStream_t st)
{
	const bool full = p.dim * (int)sizeof(T) == 32 << lg;
	if (!turn_four(p, norm, lg, (int)sizeof(T))) return full ? turn_launch<T, FORM, PART, 2, true>(p, norm, lg, st) : turn_launch<T, FORM, PART, 2, false>(p, norm, lg, st);
	return full ? turn_launch<T, FORM, PART, 4, true>(p, norm, lg, st) : turn_launch<T, FORM, PART, 4, false>(p, norm, lg, st);
}

template <class T, int FORM> static int turn_part(TurnArgs &p, bool norm, int lg, cudaStream_t st)
{
	constexpr int E = 16 / (int)sizeof(T);
	const int part = (E << lg) / 32; // pairs that a thread computes for those of its place in other rows
	return part == 4 ? turn_rounds<T, FORM, 4>(p, norm, lg, st) : part == 2 ? turn_rounds<T, FORM, 2>(p, norm, lg, st) : turn_rounds<T, FORM, 1>(p, norm, lg, st);
}

template <class T, int NI> static int turn_any(TurnArgs &p, bool norm, cudaStream_t st)
{
	const __int128 items = (__int128)p.all * p.chunks;
	const long long blocks = items > 0x1ffffffffll ? 0x80000000ll : (long long)(items + 3) / 4;
	if (turn_grid(blocks)) return TG_CUDA_EINVAL;
	if (norm) k_turn_any<T, true, NI><<<(unsigned)blocks, 128, 0, st>>>(p);
	else k_turn_any<T, false, NI><<<(unsigned)blocks, 128, 0, st>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

template <class T> static int turn_form(TurnArgs &p, int pairs, bool norm, cudaStream_t st)
{
	constexpr int E = 16 / (int)sizeof(T);
	const int items = (p.dim / E + 1) / 2;
	int lg = 0;
	while (1 << lg < items) lg++;
	if (pairs) return turn_part<T, TURN_PAIRS>(p, norm, lg, st);
	if (p.part * (int)sizeof(T) % 32 == 0) return turn_part<T, TURN_HALF>(p, norm, lg, st);
	p.chunks = 0;
	for (int g = 0; g < p.nrows; g++) p.chunks += p.rows[g].chunks = (p.rows[g].heads + TURN_ANY_ROWS - 1) / TURN_ANY_ROWS;
	return p.dim <= 64 ? turn_any<T, 1>(p, norm, st) : p.dim <= 128 ? turn_any<T, 2>(p, norm, st) : turn_any<T, 4>(p, norm, st);
}

static int turn_type(TurnArgs &p, int type, int pairs, bool norm, void *stream)
{
	cudaStream_t st = (cudaStream_t)stream;
	return type == TG_CUDA_F32 ? turn_form<float>(p, pairs, norm, st) : type == TG_CUDA_F16 ? turn_form<__half>(p, pairs, norm, st) : turn_form<__nv_bfloat16>(p, pairs, norm, st);
}

// An output's rows: on 16-byte boundaries, none over another, and those of its input (strides in[], bytes) only each in its own place.
// Strides along one element are not used.
static int turn_out(const char *who, const char *what, void *out, long long (&s)[3], const void *x, const long long (&in)[3], int seqs, int tokens, int heads, int dim, int e)
{
	const int n[3] = { seqs, tokens, heads };
	for (int i = 0; i < 3; i++) {
		if (n[i] <= 1) s[i] = 0;
		else if (out == x && s[i] * e != in[i]) return set_err(TG_CUDA_EINVAL, "%s: %s is its input with other strides", who, what);
	}
	if (((uintptr_t)out & 15) || ((s[0] | s[1] | s[2]) * e & 15)) return set_err(TG_CUDA_EINVAL, "%s: %s rows must start on 16-byte boundaries", who, what);
	return pg_apart(who, what, dim, { s[0], s[1], s[2] }, { seqs, tokens, heads });
}

// Rows that a call writes may not be rows that it reads, which other warps read at any time, nor other rows that it writes; those that
// `same` names may be it, each in its own place (turn_out has looked at the strides).
static int turn_apart(const char *who, const char *what, const PgRows &out, const PgRows &other, const char *name, bool same)
{
	if ((same && out.at == other.at) || !pg_meet(out, other)) return TG_CUDA_OK;
	return set_err(TG_CUDA_EINVAL, "%s: %s and %s share memory", who, what, name);
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
	if ((rc = turn_check(who, r, head_dim, seqs, &p))) return rc;
	const bool none = !seqs || !tokens || !heads;
	if (!none && (!x || !out)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	long long s[3] = { seqs > 1 ? x_seq : 0, tokens > 1 ? x_tok : 0, heads > 1 ? x_head : 0 }, o[3] = { out_seq, out_tok, out_head };
	if (s[0] < 0 || s[1] < 0 || s[2] < 0) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	if (((uintptr_t)x & 15) || ((s[0] | s[1] | s[2]) * e & 15)) return set_err(TG_CUDA_EINVAL, "%s: x rows must start on 16-byte boundaries", who);
	if (!none && (rc = turn_out(who, "out", out, o, x, { s[0] * e, s[1] * e, s[2] * e }, seqs, tokens, heads, head_dim, e))) return rc;
	if (!none && (rc = turn_apart(who, "out", { out, head_dim * e, { o[0] * e, o[1] * e, o[2] * e }, { seqs, tokens, heads } },
				      { x, head_dim * e, { s[0] * e, s[1] * e, s[2] * e }, { seqs, tokens, heads } }, "x", true)))
		return rc;
	if ((rc = pg_sms(who, &dev, &sms)) || none) return rc;
	p.rows[0] = { (const char *)x, (char *)out, nullptr, s[0] * e, s[1] * e, s[2] * e, o[0] * e, o[1] * e, o[2] * e, nullptr, heads, r->dim > 0, 0, 0, 0 };
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
	if (r && (rc = turn_check(who, r, c->head_dim, c->seqs, &p))) return rc;
	if (c->seqs && (!len_out || !d->q != !q_out)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if ((rc = pg_len_out(who, c, d, len_out))) return rc;
	if (((uintptr_t)len_out | (uintptr_t)q_norm | (uintptr_t)k_norm) & 3) return set_err(TG_CUDA_EINVAL, "%s: a pointer is not on a 4-byte boundary", who);
	if (q_norm && !q) return set_err(TG_CUDA_EINVAL, "%s: q_norm without q", who);
	long long qo[3] = { q_out_seq, q_out_tok, q_out_head }, ko[3] = { k_out_seq, k_out_tok, k_out_head };
	if (q && (rc = turn_out(who, "q_out", q_out, qo, pd.q, { pd.q_seq, pd.q_tok, pd.q_head }, c->seqs, d->tokens, d->nq, c->head_dim, e))) return rc;
	if (k_out && (rc = turn_out(who, "k_out", k_out, ko, pd.k, { pd.kv_seq, pd.kv_tok, pd.kv_head }, c->seqs, d->tokens, c->nkv, c->head_dim, e))) return rc;
	const long long row = c->head_dim * e;
	const PgRows rq = { q ? pd.q : nullptr, row, { pd.q_seq, pd.q_tok, pd.q_head }, { c->seqs, d->tokens, d->nq } }, rk = { pd.k, row, { pd.kv_seq, pd.kv_tok, pd.kv_head }, { c->seqs, d->tokens, c->nkv } },
		     rv = { pd.v, row, rk.stride, rk.n }, ro = { q ? q_out : nullptr, row, { qo[0] * e, qo[1] * e, qo[2] * e }, rq.n }, rl = { k_out, row, { ko[0] * e, ko[1] * e, ko[2] * e }, rk.n };
	if ((rc = turn_apart(who, "q_out", ro, rq, "q", true)) || (rc = turn_apart(who, "q_out", ro, rk, "k", false)) || (rc = turn_apart(who, "q_out", ro, rv, "v", false)) ||
	    (rc = turn_apart(who, "k_out", rl, rq, "q", false)) || (rc = turn_apart(who, "k_out", rl, rk, "k", true)) || (rc = turn_apart(who, "k_out", rl, rv, "v", false)) ||
	    (rc = turn_apart(who, "q_out", ro, rl, "k_out", false)))
		return rc;
	if ((rc = pg_apart(who, "the cache", c->head_dim, {c->page_stride, c->head_stride, c->pos_stride}, {c->pages, c->nkv, c->page}))) return rc;
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0) return rc;
	if (q) p.rows[p.nrows++] = { pd.q, (char *)q_out, nullptr, pd.q_seq, pd.q_tok, pd.q_head, qo[0] * e, qo[1] * e, qo[2] * e, q_norm, d->nq, r && r->dim, 0, !((uintptr_t)q_norm & 15), 0 };
	p.rows[p.nrows++] = { pd.k, (char *)k_out, p.c.k, pd.kv_seq, pd.kv_tok, pd.kv_head, ko[0] * e, ko[1] * e, ko[2] * e, k_norm, c->nkv, r && r->dim, 1, !((uintptr_t)k_norm & 15), 0 };
	p.rows[p.nrows++] = { pd.v, nullptr, p.c.v, pd.kv_seq, pd.kv_tok, pd.kv_head, 0, 0, 0, nullptr, c->nkv, 0, 1, 0, 0 };
	p.count = d->count, p.len_out = len_out, p.all = (long long)c->seqs * d->tokens, p.tokens = d->tokens, p.dim = c->head_dim, p.over_dim = 1.f / c->head_dim, p.eps = eps;
	return turn_type(p, c->type, r && r->interleaved, q_norm || k_norm, stream);
}
