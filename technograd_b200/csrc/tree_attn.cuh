// tree_attn.cuh -- attention of drafted tokens over a paged cache: the kernel for few query rows, and
// the join of partial results. One source per element type instantiates it (tree_attn_*.cu).
#pragma once

#include <type_traits>

#include "common.cuh"
#include "mma_sync.cuh"
#include "paged.cuh"

namespace tgc {

struct AttnArgs {
	PgCache c;
	PgDrafts d;
	char *out;
	long long out_seq, out_tok, out_head; // bytes
	float *lse;
	int seqs;
	int row_tiles;   // tiles of 16 * MT query rows per (sequence, kv head)
	int whole;       // 1: a CTA per unit; 0: equal shares of the units' tiles
	int least;       // shares: tiles per CTA at least
	int begin;       // shares: what beginning a unit costs, in tiles
	PgBox box;       // of the pools' TMA maps; rows 0: none
	float *part;     // shares: partial results, two slots per CTA
	int ctas;        // of the launch
	int by_unit;     // shares: split's entries are the units', else the CTAs'
	int4 *split;     // shares: of a unit that begins in a CTA's share and ends in a later one, the two CTAs, its
	                 // sequence and head, and its row tile; x = -1: none, or nothing to join
};

struct WeightArgs : AttnArgs { // its lse is the input; out and part are not used
	const unsigned long long *select;
	const float *acc;
	long long acc_seq, acc_head;
	float *acc_out, *fresh;
};

// Attention below shared prefixes (shared_attn.cuh) runs the kernels twice: over the groups' prefixes, whose units have the rows of
// all members, and over what each sequence has of its own. Neither writes results: what a CTA has of a unit as a whole goes to
// rows of its own, parts as above, and a join of both follows.
enum { ATTN_ALL, ATTN_PREFIX, ATTN_OWN };

struct SharedArgs : AttnArgs {
	const int *first, *members, *shared, *group;
	int groups, max_shared;
	int align;       // a prefix ends at a multiple of this, a power of two; what is left of it is the sequences' own
	float *whole_o;  // [rows][DP]: the rows of units that one CTA had, O before the division
	float2 *whole_ml; // their reference and sum
	int2 *tab;       // [units]: the first and last CTA of a unit, x = -1: one CTA had it all
	int pitch;       // prefixes: entries of tab per head

	// Sequence b's positions n, and how many of them it shares with its group g (-1: none). The length and the group are read at
	// once: each further load in a row would be another half of a microsecond before a unit begins.
	__device__ __forceinline__ int from(int b, int &n, int &g) const
	{
		const int len = c.len[b];
		g = group[b];
		const bool in = (unsigned)g < (unsigned)groups;
		const int s = in ? shared[g] : 0;
		if (len < 0 || len > c.max_len) c.report(PG_LEN);
		n = max(0, min(len, c.max_len));
		if (s < 0 || s > max_shared || s > n || (!in && g != -1)) c.report(PG_GROUP);
		if (!in) g = -1;
		return max(0, min(s, min(n, max_shared))) & -align;
	}
	// the sequences of group g and their shared positions
	__device__ __forceinline__ void prefix(int g, int &seq, int &m, int &n) const
	{
		const int f = first[g], k = members[g];
		if (f < 0 || k < 0 || f > seqs || k > seqs - f) c.report(PG_GROUP);
		seq = max(0, min(f, seqs)), m = max(0, min(k, seqs - seq));
		n = m == 0 ? 0 : max(0, min(shared[g], min(max_shared, c.length(seq)))) & -align;
	}
	// place of a prefix's first unit in a head's part of tab: groups follow one another, so that no two meet
	__device__ __forceinline__ long long base(int g, int seq, int rt) const { return (long long)seq * d.tokens * d.group / rt + g; }
};
template <int MODE> using AttnArgsOf = std::conditional_t<MODE == ATTN_ALL, AttnArgs, SharedArgs>;

// exp(scale s - lse). The difference is taken before anything is multiplied by log2(e): of a key with much weight it is
// near 0, while scale s and lse may be tens, and their products' roundings would be errors of 1e-6 in the weight.
__device__ __forceinline__ float weight_of(float s, float scale, float lse) { return ex2(fmaf(s, scale, -lse) * 1.4426950408889634f); }

// The kernel for few query rows. Per (sequence b, kv head h) the query rows are r = t * group + g
// (token t, query head h * group + g): every head of the group and every drafted token meet a key
// while it is in shared memory, so the cache is read once for up to 16 * MT rows.
//
// Unit = (b, h, tile of 16 * MT rows); its keys are the cached positions in tiles of 4 * KW, then the
// drafted tokens in as many tiles as they need. A CTA's four warps each take KW keys of a tile and
// work on their own: a ring of NST stages of cp.async copies per warp (K and V rows, XOR-swizzled),
// S = Q K^T on the tensor cores, p = 2^(z - mr) with z = scale log2(e) s, and O += P V with O in
// registers. mr is a running reference for each row, raised (O and l rescaled) only when a score
// exceeds it by RAISE, so the usual step needs no maximum across lanes; p stays below 2^(RAISE + SHIFT)
// and the quotient O / l is the softmax's whatever mr is. At a unit's end the four warps' O are
// brought to one reference and summed in warp order through the stage each of them has free.
//
// What bounds it: the cache's bytes. Lengths differ and units are few or many, so the CTAs of one
// wave take equal shares of all units' tiles, in order; the ring runs on across unit boundaries. A
// unit that ends in its CTA's share is written out; of one that spans several, each CTA leaves
// (O, mr, l), and k_attn_join adds them in CTA order: results do not depend on timing.
// Measured: a decode wave of 256 sequences of up to 1280 positions (16 query heads over 8, 128 dimensions, bf16) 183 us
// in a stream of calls, 5.4 TB/s (167 in the first few hundred, before the card is at its power limit).
template <class T> struct AttnScale; // SHIFT: exponent given to probabilities near 1
template <> struct AttnScale<float> { static constexpr float SHIFT = 0, RAISE = 8; };
template <> struct AttnScale<__nv_bfloat16> { static constexpr float SHIFT = 0, RAISE = 8; };
// f16 has 5 exponent bits: probabilities from 2^-24 to 2^5 of the reference must be normal numbers
template <> struct AttnScale<__half> { static constexpr float SHIFT = 10, RAISE = 5; };

template <class T, int DP, int MT> struct AttnTile {
	static constexpr int KW = sizeof(T) == 4 ? 8 : 16, NT = KW / 8, TK = 4 * KW, RT = 16 * MT;
	static constexpr int P = DP * (int)sizeof(T), CH = P / 16;
	static constexpr int STAGE = 2 * KW * P; // also 16 x DP floats, what the end of a unit needs
	// 16 rows of 16-bit elements: three CTAs per SM with a stage ahead each, 183 us for a 256-sequence decode wave
	// against 195 of two CTAs with two ahead; the others' registers allow two
	static constexpr int CTAS = DP == 256 ? 1 : MT == 1 && sizeof(T) == 2 ? 3 : 2;
	static constexpr int NST = CTAS == 3 || DP == 256 || (DP == 128 && MT == 2 && sizeof(T) == 4) ? 2 : 3;
	static constexpr int Q = 0, QLO = RT * P, RING = sizeof(T) == 4 ? 2 * QLO : QLO, MASK = RING + 4 * NST * STAGE, ML = MASK + RT * 8, SCAN = ML + 4 * RT * 8; // QLO: Q's low parts, f32
	static constexpr int SMEM = SCAN + 128; // attn_share: 2 * 4 + 6 words
	static constexpr int SLOT = RT * DP + 2 * RT; // floats of a partial result
};

// A place in the list of tiles.
struct AttnCursor {
	int b, h, r, tile, ctx, n, all; // ctx: tiles of cached positions, all: with the drafted ones
	int p0;                         // own positions: the first of them
	int seq, rows, tiles;           // prefixes (b: the group): the first member, the unit's rows and row tiles
};

template <int TK, int MODE = ATTN_ALL, int RT = 1>
__device__ __forceinline__ void cursor_seq(const AttnArgsOf<MODE> &p, AttnCursor &c, int extra)
{
	if constexpr (MODE == ATTN_PREFIX) {
		int m;
		p.prefix(c.b, c.seq, m, c.n);
		c.rows = m * p.d.tokens * p.d.group, c.tiles = (c.rows + RT - 1) / RT;
		c.ctx = c.all = (int)(((long long)c.n + TK - 1) / TK);
	} else {
		if constexpr (MODE == ATTN_OWN) {
			int g;
			c.p0 = p.from(c.b, c.n, g);
			c.ctx = (int)(((long long)c.n - c.p0 + TK - 1) / TK);
		} else {
			c.n = p.c.length(c.b);
			c.ctx = (int)(((long long)c.n + TK - 1) / TK);
		}
		c.all = c.ctx + extra;
	}
}

template <int TK, int MODE = ATTN_ALL, int RT = 1>
__device__ __forceinline__ void cursor_next(const AttnArgsOf<MODE> &p, AttnCursor &c, int extra)
{
	if (++c.tile < c.all) return;
	c.tile = 0;
	if (++c.r < (MODE == ATTN_PREFIX ? c.tiles : p.row_tiles)) return;
	c.r = 0;
	if (++c.h < p.c.nkv) return;
	c.h = 0;
	if constexpr (MODE == ATTN_PREFIX) {
		while (++c.b < p.groups) {
			cursor_seq<TK, MODE, RT>(p, c, extra);
			if (c.all) break;
		}
	} else if (++c.b < p.seqs) cursor_seq<TK, MODE, RT>(p, c, extra);
}

// Sum of a value over the CTA's NW warps, and the sum over the threads before this one.
template <int NW>
__device__ __forceinline__ long long block_scan(long long v, long long *s, long long &before)
{
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	long long x = v;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const long long y = __shfl_up_sync(~0u, x, o);
		if (lane >= o) x += y;
	}
	__syncthreads();
	if (lane == 31) s[warp] = x;
	__syncthreads();
	before = x - v;
	long long all = 0;
#pragma unroll
	for (int w = 0; w < NW; w++) {
		if (w < warp) before += s[w];
		all += s[w];
	}
	return all;
}

// a / b of numbers that nearly always fit 32 bits (a 64-bit division is a long chain of instructions)
__device__ __forceinline__ long long quotient(long long a, unsigned b) { return a >> 32 ? a / b : (long long)((unsigned)a / b); }

// What a CTA works on: `left` tiles from place c of the list. s: NW + 4 words of shared memory, for prefixes 2 NW + 6.
// False: nothing. A unit counts its tiles and p.begin more, spent before its first tile; the CTAs' shares of
// the total are equal, share and pos being one's size and beginning.
template <int TK, int NW, int MODE = ATTN_ALL, int RT = 1>
__device__ __forceinline__ bool attn_share(const AttnArgsOf<MODE> &p, long long *s, int extra, AttnCursor &c, long long &left, long long &pos, long long &share)
{
	if (p.whole) {
		c.r = blockIdx.x % p.row_tiles;
		c.h = blockIdx.x / p.row_tiles % p.c.nkv;
		c.b = blockIdx.x / p.row_tiles / p.c.nkv;
		c.tile = 0;
		cursor_seq<TK, MODE, RT>(p, c, extra);
		left = c.all, pos = 0, share = 1;
		return true;
	}
	const int per = p.c.nkv * p.row_tiles, lists = MODE == ATTN_PREFIX ? ((const SharedArgs &)p).groups : p.seqs;
	auto units = [&](int b) -> long long { // prefixes
		AttnCursor x;
		x.b = b;
		if (b >= lists) return 0;
		cursor_seq<TK, MODE, RT>(p, x, extra);
		return x.all ? (long long)x.tiles * p.c.nkv : 0;
	};
	auto weight = [&](int b) -> long long {
		if constexpr (MODE == ATTN_ALL) return b < p.seqs ? (((long long)p.c.length(b) + TK - 1) / TK + extra + p.begin) * per : 0;
		else {
			AttnCursor x;
			x.b = b;
			if (b >= lists) return 0;
			cursor_seq<TK, MODE, RT>(p, x, extra);
			return MODE == ATTN_OWN ? ((long long)x.all + p.begin) * per : x.all ? ((long long)x.all + p.begin) * p.c.nkv * x.tiles : 0;
		}
	};
	const bool once = lists <= 32 * NW; // a thread per sequence: one pass over the lengths
	long long mine = 0, before, all;
	for (int b = threadIdx.x; b < lists; b += 32 * NW) mine += weight(b);
	all = block_scan<NW>(mine, s, before);
	share = quotient(all + gridDim.x - 1, gridDim.x);
	if (share < p.least + p.begin) share = p.least + p.begin;
	pos = share * blockIdx.x;
	if (MODE == ATTN_ALL && threadIdx.x == 0 && p.split && !p.by_unit) p.split[blockIdx.x].x = -1;
	if (pos >= all) return false;
	const long long to = all - pos < share ? all : pos + share; // the place after the share
	long long base = 0;
	long long *su = s + NW + 4; // prefixes: the units before the two places
	long long ubase = 0, ubefore = 0;
	for (int b0 = 0;; b0 += 32 * NW) { // ends: pos < to <= all
		const int b = b0 + threadIdx.x;
		const long long w = once ? mine : weight(b), sum = once ? all : block_scan<NW>(w, s, before);
		long long usum = 0;
		if constexpr (MODE == ATTN_PREFIX) usum = block_scan<NW>(units(b), su, ubefore);
		if (pos >= base + before && pos < base + before + w) {
			s[NW] = b, s[NW + 1] = base + before;
			if constexpr (MODE == ATTN_PREFIX) su[NW] = ubase + ubefore;
		}
		if (to - 1 >= base + before && to - 1 < base + before + w) {
			s[NW + 2] = b, s[NW + 3] = base + before;
			if constexpr (MODE == ATTN_PREFIX) su[NW + 1] = ubase + ubefore;
		}
		base += sum, ubase += usum;
		if (to <= base) break;
	}
	__syncthreads();
	// tiles before the place `off` into sequence b's units, whose units begin at place `first`
	int u, t, in;
	auto tiles = [&](long long b, long long first, long long off, long long before) {
		c.b = (int)b;
		cursor_seq<TK, MODE, RT>(p, c, extra);
		u = (int)quotient(off, c.all + p.begin);
		in = (int)(off - (long long)u * (c.all + p.begin));
		t = in < p.begin ? 0 : in - p.begin;
		return first - (MODE == ATTN_PREFIX ? before : b * per) * p.begin + (long long)u * c.all + t;
	};
	left = tiles(s[NW + 2], s[NW + 3], to - 1 - s[NW + 3], MODE == ATTN_PREFIX ? su[NW + 1] : 0);
	if (in >= p.begin) left++; // the last place is a tile's
	left -= tiles(s[NW], s[NW + 1], pos - s[NW + 1], MODE == ATTN_PREFIX ? su[NW] : 0);
	const int rt = MODE == ATTN_PREFIX ? c.tiles : p.row_tiles;
	c.tile = t, c.h = u / rt, c.r = u % rt;
	return left > 0;
}

// Notes, at the end of the part of a unit that has its first tile, whether other CTAs have the rest. c: the part's last tile.
__device__ __forceinline__ void attn_note(const AttnArgs &p, const AttnCursor &c, bool whole, long long pos, long long share)
{
	if (p.whole || (whole && !p.by_unit)) return;
	const int head = c.b * p.c.nkv + c.h;
	p.split[p.by_unit ? (long long)head * p.row_tiles + c.r : blockIdx.x] =
		whole ? make_int4(-1, 0, 0, 0) : make_int4(blockIdx.x, (int)((pos + share + (c.all - 2 - c.tile)) / share), head, c.r);
}

// The same in a table of all units. (An entry out of its bounds: lists of groups that overlap, which are reported.)
template <int MODE, int RT>
__device__ __forceinline__ void shared_note(const SharedArgs &p, const AttnCursor &c, bool whole, long long pos, long long share)
{
	const long long at = MODE == ATTN_PREFIX ? p.base(c.b, c.seq, RT) + c.r : ((long long)c.b * p.c.nkv + c.h) * p.row_tiles + c.r;
	if (MODE == ATTN_PREFIX && at >= p.pitch) return;
	p.tab[MODE == ATTN_PREFIX ? (long long)c.h * p.pitch + at : at] =
		whole ? make_int2(-1, -1) : make_int2(blockIdx.x, (int)((pos + share + (c.all - 2 - c.tile)) / share));
}

// Row r of a unit: its sequence, token and query head.
struct SharedRow {
	int b, t, j;
};
template <int MODE> __device__ __forceinline__ SharedRow shared_row(const AttnArgs &p, const AttnCursor &c, int r)
{
	const int x = r / p.d.group, j = c.h * p.d.group + (r - x * p.d.group);
	if constexpr (MODE != ATTN_PREFIX) return { c.b, x, j };
	const int m = x / p.d.tokens;
	return { c.seq + m, x - m * p.d.tokens, j };
}
__device__ __forceinline__ const char *q_row(const AttnArgs &p, SharedRow x) { return p.d.q + x.b * p.d.q_seq + x.t * p.d.q_tok + x.j * p.d.q_head; }
__device__ __forceinline__ long long whole_row(const AttnArgs &p, SharedRow x) { return ((long long)x.b * p.d.tokens + x.t) * p.d.nq + x.j; }

// The two passes and their join follow one another without a gap: the pass over own positions begins as soon as the prefixes' CTAs
// leave room. Those have waited for what came before the call, and a grid counts as launched when all its CTAs have, so that
// nothing before the call runs any more; and the own positions' CTAs end after the prefixes', so that the join
// finds both.
template <int MODE> __device__ __forceinline__ void shared_begin()
{
	if (MODE == ATTN_PREFIX) pdl_wait();
	pdl_launch();
}
template <int MODE> __device__ __forceinline__ void shared_end()
{
	if (MODE == ATTN_OWN) pdl_wait();
}

// A partial result's place of 4 columns of a row (then come the rows' mr and l): as the kernel that
// leaves it writes whole lines, a row's columns together from k_tree_attn, the rows of 4 columns together
// from the row per thread of the tiles of 128 rows and more.
template <int DP, int RT> __device__ __forceinline__ int slot_at(int row, int col) { return RT >= 128 ? (col / 4 * RT + row) * 4 : row * DP + col; }

// o (already over l, or a partial's) of 4 columns
__device__ __forceinline__ void store4(float *d, float4 v) { *(float4 *)d = v; }
__device__ __forceinline__ void store4(__half *d, float4 v) { *(uint2 *)d = make_uint2(pack16(v.x, v.y, __half()), pack16(v.z, v.w, __half())); }
__device__ __forceinline__ void store4(__nv_bfloat16 *d, float4 v)
{
	*(uint2 *)d = make_uint2(pack16(v.x, v.y, __nv_bfloat16()), pack16(v.z, v.w, __nv_bfloat16()));
}

// Where a row's result goes, and what it is divided by: a token past the count, or one that saw nothing, has
// 0 and -infinity.
struct AttnRow {
	char *out;
	float *lse;
	float f; // 1 / l, 0 for none
	bool none;
};
__device__ __forceinline__ AttnRow attn_row(const AttnArgs &p, int b, int h, int row, int cnt, float l)
{
	const int t = row / p.d.group, j = h * p.d.group + (row - t * p.d.group);
	AttnRow x;
	x.out = p.out + b * p.out_seq + t * p.out_tok + j * p.out_head;
	x.lse = p.lse + ((long long)b * p.d.tokens + t) * p.d.nq + j;
	x.none = t >= cnt || l == 0;
	x.f = x.none ? 0 : 1 / l;
	return x;
}
__device__ __forceinline__ void store_lse(const AttnRow &x, float mr, float l) { *x.lse = x.none ? -INFINITY : (mr + log2f(l)) * 0.69314718056f; }
// 8 columns of a row: whole 16-byte pieces for 16-bit elements
template <class T>
__device__ __forceinline__ void store_row8(const AttnArgs &p, const AttnRow &x, int col, const float *o)
{
	if (col >= p.c.dim) return;
	float v[8];
#pragma unroll
	for (int i = 0; i < 8; i++) v[i] = x.none ? 0 : o[i] * x.f;
	if constexpr (sizeof(T) == 2)
		*(uint4 *)((T *)x.out + col) = make_uint4(pack16(v[0], v[1], T()), pack16(v[2], v[3], T()), pack16(v[4], v[5], T()), pack16(v[6], v[7], T()));
	else {
		store4((T *)x.out + col, make_float4(v[0], v[1], v[2], v[3]));
		if (col + 4 < p.c.dim) store4((T *)x.out + col + 4, make_float4(v[4], v[5], v[6], v[7]));
	}
}
template <class T>
__device__ __forceinline__ void store_row4(const AttnArgs &p, const AttnRow &x, int col, float4 o)
{
	if (col >= p.c.dim) return;
	if (x.none) o = make_float4(0, 0, 0, 0);
	store4((T *)x.out + col, make_float4(o.x * x.f, o.y * x.f, o.z * x.f, o.w * x.f));
}

// A warp's fetching of its rows of the tiles to come, K and V: lane i < KW holds the place of the tile's row i, looked up
// while the tile before is fetched.
template <class T, int DP, class A, int MODE = ATTN_ALL> struct AttnFetch {
	const AttnArgsOf<MODE> &p;
	AttnCursor f;
	long long left, fetched = 0;
	uint32_t at = PG_NONE, ring;
	int extra, chunks;

	__device__ __forceinline__ AttnFetch(const AttnArgsOf<MODE> &args, const AttnCursor &c, long long n, uint32_t stages, int drafted_tiles, int row_chunks)
		: p(args), f(c), left(n), ring(stages), extra(drafted_tiles), chunks(row_chunks)
	{
		find();
	}
	__device__ __forceinline__ void find()
	{
		const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
		at = PG_NONE;
		if (lane >= A::KW || fetched >= left) return;
		if (f.tile < f.ctx) {
			const int x = (MODE == ATTN_OWN ? f.p0 : 0) + f.tile * A::TK + warp * A::KW + lane;
			if (x < f.n) {
				const int page = x / p.c.page;
				at = p.c.at(p.c.table[(long long)(MODE == ATTN_PREFIX ? f.seq : f.b) * p.c.cols + page], x - page * p.c.page);
			}
		} else {
			const int u = (f.tile - f.ctx) * A::TK + warp * A::KW + lane;
			if (u < p.d.drafted(f.b)) at = (uint32_t)(u * p.d.kv_tok >> 4);
		}
	}
	// the next tile, if there is one, into a stage; always one group of copies
	__device__ __forceinline__ void fetch(int stage)
	{
		if (fetched < left) {
			const int lane = threadIdx.x & 31;
			const bool ctx = f.tile < f.ctx;
			const int sh = ctx ? p.c.shift : 4;
			const long long head = ctx ? f.h * p.c.head_b : f.b * p.d.kv_seq + f.h * p.d.kv_head;
			const char *kp = (ctx ? p.c.k : p.d.k) + head, *vp = (ctx ? p.c.v : p.d.v) + head;
			const uint32_t sk = ring + stage * A::STAGE, sv = sk + A::KW * A::P, mine = at;
			cursor_next<A::TK, MODE, A::RT>(p, f, extra);
			fetched++;
			find();
#pragma unroll
			for (int i = 0; i < A::KW * A::CH / 32; i++) {
				const int row = (i * 32 + lane) / A::CH, ch = (i * 32 + lane) % A::CH;
				const uint32_t r = __shfl_sync(~0u, mine, row), o = row * A::P + ((ch ^ (row & 7)) << 4);
				const bool have = r != PG_NONE && ch < chunks;
				const unsigned long long off = ((unsigned long long)r << sh) + ch * 16;
				cp16(sk + o, have ? kp + off : p.d.k, have);
				cp16(sv + o, have ? vp + off : p.d.v, have);
			}
		}
		cp_commit();
	}
};

template <class T, int DP, int MT, int MODE = ATTN_ALL>
__global__ void __launch_bounds__(128, AttnTile<T, DP, MT>::CTAS) k_tree_attn(const AttnArgsOf<MODE> p)
{
	using A = AttnTile<T, DP, MT>;
	constexpr int KW = A::KW, NT = A::NT, TK = A::TK, RT = A::RT, P = A::P, CH = A::CH, NST = A::NST;
	constexpr float SHIFT = AttnScale<T>::SHIFT, RAISE = AttnScale<T>::RAISE;
	extern __shared__ __align__(128) char smem[];
	unsigned long long *s_mask = (unsigned long long *)(smem + A::MASK);
	float2 *s_ml = (float2 *)(smem + A::ML);
	long long *s_scan = (long long *)(smem + A::SCAN);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
	const uint32_t s0 = smem_u32(smem), ring = s0 + A::RING + warp * NST * A::STAGE;
	const int extra = MODE == ATTN_PREFIX ? 0 : (p.d.tokens + TK - 1) / TK, chunks = p.c.dim * (int)sizeof(T) / 16;
	int rows = p.d.tokens * p.d.group;
	const bool twin = MT == 1 && sizeof(T) == 2 && MODE != ATTN_PREFIX && rows <= 8; // rows 8 to 15 are rows 0 to 7 again (pv_tile)
	const float zs = p.d.scale * 1.4426950408889634f;
	if constexpr (MODE == ATTN_ALL) {
		pdl_launch();
		pdl_wait();
	} else shared_begin<MODE>();

	AttnCursor c; // the tile being worked on; f, below: the next to be fetched
	long long left, pos, share;
	if (!attn_share<TK, 4, MODE, RT>(p, s_scan, extra, c, left, pos, share)) {
		shared_end<MODE>();
		return;
	}

	AttnFetch<T, DP, A, MODE> f(p, c, left, ring, extra, chunks);
	auto fetch = [&](int stage) { f.fetch(stage); };

	float o[MT][DP / 8][4], mr[MT][2], l[MT][2];
	int cnt = 0;
	bool first = true, from_start = true; // from_start: this CTA has the unit's first tile
	int stage = 0;
#pragma unroll
	for (int i = 0; i < NST - 1; i++) fetch(i);

	for (long long i = 0; i < left; i++) {
		if (first) { // a unit begins here, or goes on from the CTA before
			first = false;
			from_start = c.tile == 0;
			if constexpr (MODE == ATTN_PREFIX) rows = c.rows;
			else cnt = p.d.drafted(c.b);
			for (int x = tid; x < RT * CH; x += 128) {
				const int row = x / CH, ch = x % CH, r = c.r * RT + (twin ? row & 7 : row), t = r / p.d.group;
				uint4 v = make_uint4(0, 0, 0, 0);
				if (r < rows && ch < chunks) {
					if constexpr (MODE == ATTN_PREFIX) v = *(const uint4 *)(q_row(p, shared_row<MODE>(p, c, r)) + ch * 16);
					else v = *(const uint4 *)(p.d.q + (long long)c.b * p.d.q_seq + (long long)t * p.d.q_tok + (long long)(c.h * p.d.group + r % p.d.group) * p.d.q_head + ch * 16);
				}
				*(uint4 *)(smem + row * P + ((ch ^ (row & 7)) << 4)) = v;
				if constexpr (sizeof(T) == 4) *(uint4 *)(smem + A::QLO + row * P + ((ch ^ (row & 7)) << 4)) = tf32_low(v);
			}
			if (MODE != ATTN_PREFIX && tid < RT) {
				const int t = (c.r * RT + (twin ? tid & 7 : tid)) / p.d.group;
				s_mask[tid] = t < cnt ? p.d.sees(c.b, t, cnt) : 0;
			}
#pragma unroll
			for (int m = 0; m < MT; m++) {
				mr[m][0] = mr[m][1] = -INFINITY, l[m][0] = l[m][1] = 0;
#pragma unroll
				for (int d = 0; d < DP / 8; d++) o[m][d][0] = o[m][d][1] = o[m][d][2] = o[m][d][3] = 0;
			}
			__syncthreads();
		}
		fetch((stage + NST - 1) % NST); // into the stage of the tile before
		cp_wait<NST - 1>();
		__syncwarp();
		const uint32_t sk = ring + stage * A::STAGE, sv = sk + KW * P;
		const bool drafted = c.tile >= c.ctx;
		float s[MT][NT][4];
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++) s[m][x][0] = s[m][x][1] = s[m][x][2] = s[m][x][3] = 0;
		qk_tile<T, DP, MT, NT>(s, s0, sk, lane, A::QLO);
		unsplit_scores<T, DP, MT, NT>(s, s0, sk, lane);
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++)
#pragma unroll
				for (int e = 0; e < 4; e++) s[m][x][e] *= zs;
		if (drafted || c.tile == c.ctx - 1) { // the mask's bits, or the end of the cache
			const long long at = (long long)(drafted ? c.tile - c.ctx : c.tile) * TK + warp * KW + (MODE == ATTN_OWN && !drafted ? c.p0 : 0);
#pragma unroll
			for (int m = 0; m < MT; m++)
#pragma unroll
				for (int x = 0; x < NT; x++)
#pragma unroll
					for (int e = 0; e < 4; e++) {
						const long long key = at + x * 8 + 2 * t4 + (e & 1);
						const bool ok = drafted ? s_mask[m * 16 + g + (e >> 1) * 8] >> key & 1 : key < c.n;
						if (!ok) s[m][x][e] = -INFINITY;
					}
		}
		// raise the references?
		bool up = false;
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int x = 0; x < NT; x++)
#pragma unroll
				for (int e = 0; e < 4; e++) up |= s[m][x][e] > mr[m][e >> 1] + (SHIFT + RAISE);
		if (__any_sync(~0u, up)) {
#pragma unroll
			for (int m = 0; m < MT; m++)
#pragma unroll
				for (int e = 0; e < 2; e++) {
					float top = s[m][0][2 * e];
#pragma unroll
					for (int x = 0; x < NT; x++) top = fmaxf(top, fmaxf(s[m][x][2 * e], s[m][x][2 * e + 1]));
					top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
					top = fmaxf(top, __shfl_xor_sync(~0u, top, 2)) - SHIFT;
					if (top > mr[m][e]) {
						const float a = ex2(mr[m][e] - top);
						mr[m][e] = top, l[m][e] *= a;
#pragma unroll
						for (int d = 0; d < DP / 8; d++) // (what has lost its weight may be infinite)
							o[m][d][2 * e] = a == 0 ? 0 : o[m][d][2 * e] * a, o[m][d][2 * e + 1] = a == 0 ? 0 : o[m][d][2 * e + 1] * a;
					}
				}
		}
#pragma unroll
		for (int m = 0; m < MT; m++)
#pragma unroll
			for (int e = 0; e < 2; e++) {
				const float ref = mr[m][e] == -INFINITY ? 0 : mr[m][e]; // nothing seen yet: 2^-infinity
#pragma unroll
				for (int x = 0; x < NT; x++)
#pragma unroll
					for (int y = 2 * e; y < 2 * e + 2; y++) l[m][e] += s[m][x][y] = ex2(s[m][x][y] - ref);
			}
		bool plain = true;
		if (drafted) { // a row that some token does not see may hold anything: 0 * infinity must not reach O
			bool odd = false;
			for (int x = lane; x < KW * CH; x += 32) {
				const uint4 v = *(const uint4 *)(smem + (sv - s0) + x * 16);
				const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
				for (int y = 0; y < 4; y++) odd |= PgElem<T>::odd(w[y]);
			}
			plain = !__any_sync(~0u, odd);
		}
		if (plain) pv_tile<T, DP, MT, NT>(o, s, sv, lane, twin);
		else {
#pragma unroll
			for (int x = 0; x < NT; x++)
				for (int kk = 0; kk < 4; kk++) // the four lanes that hold keys 2 kk and 2 kk + 1
#pragma unroll
					for (int y = 0; y < 2; y++) {
						const int key = x * 8 + kk * 2 + y;
						float pr[MT][2];
#pragma unroll
						for (int m = 0; m < MT; m++)
#pragma unroll
							for (int e = 0; e < 2; e++) pr[m][e] = __shfl_sync(~0u, s[m][x][2 * e + y], (lane & ~3) | kk);
#pragma unroll
						for (int d = 0; d < DP / 8; d++)
#pragma unroll
							for (int z = 0; z < 2; z++) {
								const int col = (d * 8 + 2 * t4 + z) * (int)sizeof(T);
								const float v = PgElem<T>::get(*(const T *)(smem + (sv - s0) + key * P + (((col >> 4) ^ (key & 7)) << 4) + (col & 15)));
#pragma unroll
								for (int m = 0; m < MT; m++)
#pragma unroll
									for (int e = 0; e < 2; e++)
										if (pr[m][e] != 0 && !(twin && e)) o[m][d][2 * e + z] += pr[m][e] * v;
							}
					}
		}
		const bool end = c.tile == c.all - 1, last = i == left - 1;
		if (end || last) {
			// ---- the unit's end, or the share's: join the four warps
			if (twin) {
#pragma unroll
				for (int d = 0; d < DP / 8; d++) o[0][d][0] += o[0][d][2], o[0][d][1] += o[0][d][3];
			}
#pragma unroll
			for (int m = 0; m < MT; m++)
#pragma unroll
				for (int e = 0; e < 2; e++) {
					l[m][e] += __shfl_xor_sync(~0u, l[m][e], 1);
					l[m][e] += __shfl_xor_sync(~0u, l[m][e], 2);
					if (t4 == 0) s_ml[warp * RT + m * 16 + e * 8 + g] = make_float2(mr[m][e], l[m][e]);
				}
			__syncthreads();
			const bool complete = end && from_start;
			float *slot = complete ? nullptr : p.part + (2ll * blockIdx.x + (from_start ? 1 : 0)) * A::SLOT;
			const int b = c.b, h = c.h, r0 = c.r * RT;
#pragma unroll
			for (int m = 0; m < MT; m++) {
				float *mine = (float *)(smem + (sk - s0)); // the stage just worked on
#pragma unroll
				for (int e = 0; e < 2; e++) {
					const int row = e * 8 + g;
					float top = -INFINITY;
#pragma unroll
					for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w * RT + m * 16 + row].x);
					const float a = mr[m][e] == -INFINITY ? 0 : ex2(mr[m][e] - top);
#pragma unroll
					for (int d = 0; d < DP / 8; d++)
						*(float2 *)(mine + row * DP + ((d * 8) ^ (g * 8)) + 2 * t4) = make_float2(a == 0 ? 0 : o[m][d][2 * e] * a, a == 0 ? 0 : o[m][d][2 * e + 1] * a);
				}
				__syncthreads();
				for (int x = tid; x < 16 * DP / 4; x += 128) {
					const int row = x / (DP / 4), col = x % (DP / 4) * 4, r = m * 16 + row;
					float top = -INFINITY, sum = 0;
#pragma unroll
					for (int w = 0; w < 4; w++) top = fmaxf(top, s_ml[w * RT + r].x);
					float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
					for (int w = 0; w < 4; w++) {
						const float2 ml = s_ml[w * RT + r];
						sum += ml.x == -INFINITY ? ml.y : ml.y * ex2(ml.x - top);
						const float4 y = *(const float4 *)(smem + (ring - s0) + ((w - warp) * NST + stage) * A::STAGE + (row * DP + (col ^ ((row & 7) * 8))) * 4);
						v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
					}
					if (MODE != ATTN_ALL && complete) {
						if (r0 + r < rows) {
							const SharedArgs &sp = (const SharedArgs &)p;
							const long long to = whole_row(p, shared_row<MODE>(p, c, r0 + r));
							*(float4 *)(sp.whole_o + to * DP + col) = v;
							if (col == 0) sp.whole_ml[to] = make_float2(top, sum);
						}
					} else if (complete) {
						if (r0 + r < rows) {
							const AttnRow to = attn_row(p, b, h, r0 + r, cnt, sum);
							store_row4<T>(p, to, col, v);
							if (col == 0) store_lse(to, top, sum);
						}
					} else {
						*(float4 *)(slot + r * DP + col) = v;
						if (col == 0) slot[RT * DP + r] = top, slot[RT * DP + RT + r] = sum;
					}
				}
				__syncthreads();
			}
			if (from_start && tid == 0) {
				if constexpr (MODE == ATTN_ALL) attn_note(p, c, end, pos, share);
				else shared_note<MODE, RT>(p, c, end, pos, share);
			}
			first = true;
		}
		__syncwarp(); // every lane is done with this stage
		stage = (stage + 1) % NST;
		cursor_next<TK, MODE, RT>(p, c, extra);
	}
	cp_wait<0>();
	shared_end<MODE>();
}

// The parts of the units that several CTAs shared. A thread has a row and 8 of its columns, and the threads of a
// warp what lies together in a part; the NG warps of a block take the parts in turn (each with a running
// reference), and the first adds up what they have, in their order. Many parts (one long sequence) would be a
// chain of loads for one warp: 37 parts took it 28 us.
template <class T, int DP, int RT, int NG>
__global__ void __launch_bounds__(32 * NG) k_attn_join(const AttnArgs p)
{
	constexpr int SLOT = RT * DP + 2 * RT, RW = RT == 128 ? 32 : 1; // rows side by side in a warp
	__shared__ float s[NG > 1 ? NG : 1][10][32];
	pdl_launch();
	pdl_wait();
	const int4 u = p.split[blockIdx.x];
	// (after a wait that gave up the entry may not have been written)
	if (u.x < 0 || u.y < u.x || u.y >= p.ctas || u.z < 0 || u.z / p.c.nkv >= p.seqs || u.w < 0 || u.w >= p.row_tiles) return;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = u.z / p.c.nkv, h = u.z - b * p.c.nkv;
	const int rows = p.d.tokens * p.d.group, cnt = p.d.drafted(b), parts = u.y - u.x + 1;
	const int x = blockIdx.y * 32 + lane, r = x / (RW * DP / 8) * RW + x % RW, col = x / RW % (DP / 8) * 8;
	// nothing of the block's rows is there (a warp has 32 rows, or at 256, 128 and 64 dimensions one, two and four): the whole block
	// leaves, since single lanes may not miss its barrier
	if (u.w * RT + blockIdx.y * 32 / (RW * DP / 8) * RW >= rows) return;
	float top = -INFINITY, l = 0, v[8] = {};
	auto add = [&](float m, float n, const float *y) {
		const float t = fmaxf(top, m), f = top == -INFINITY ? 0 : ex2(top - t), a = m == -INFINITY ? 0 : ex2(m - t);
		l = (top == -INFINITY ? l : l * f) + (m == -INFINITY ? n : n * a); // sums keep a NaN
#pragma unroll
		for (int i = 0; i < 8; i++) v[i] = (f == 0 ? 0 : v[i] * f) + (a == 0 ? 0 : y[i] * a);
		top = t;
	};
#pragma unroll 4
	for (int i = warp; i < parts; i += NG) {
		const float *q = p.part + (2ll * (u.x + i) + (i == 0)) * SLOT;
		const float4 y = *(const float4 *)(q + slot_at<DP, RT>(r, col)), z = *(const float4 *)(q + slot_at<DP, RT>(r, col + 4));
		const float w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
		add(q[RT * DP + r], q[RT * DP + RT + r], w);
	}
	if constexpr (NG > 1) {
		if (warp) {
			s[warp][8][lane] = top, s[warp][9][lane] = l;
#pragma unroll
			for (int i = 0; i < 8; i++) s[warp][i][lane] = v[i];
		}
		__syncthreads();
		if (warp) return;
		for (int g = 1; g < NG && g < parts; g++) {
			float w[8];
#pragma unroll
			for (int i = 0; i < 8; i++) w[i] = s[g][i][lane];
			add(s[g][8][lane], s[g][9][lane], w);
		}
	}
	if (u.w * RT + r >= rows) return;
	const AttnRow to = attn_row(p, b, h, u.w * RT + r, cnt, l);
	store_row8<T>(p, to, col, v);
	if (col == 0) store_lse(to, top, l);
}

// How a call is cut.
struct AttnPlan {
	int dp, mt, row_tiles, whole, least, begin, grid, wave, by_unit, units, sms, dev, tc, fma; // wave: CTAs that run at once; fma: rows of tree_attn_fma.cuh, 0: another kernel; mt: 16-row products of a tile; tc: 128-row tiles on tcgen05
	size_t slot; // bytes of a partial result
	size_t bytes() const { return whole ? 0 : (size_t)grid * (2 * slot + sizeof(int4)); }
};

// tree_attn.cu: the cut of a call whose sequences have at most c->max_len positions; wide: 128-row tiles may be taken.
int attn_plan(const char *who, const tg_cuda_kv *c, const PgDrafts &d, AttnPlan *o, bool wide = true);

// Launches a planned call; T is the element type.
template <class T> int attn_type(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st);

} // namespace tgc
