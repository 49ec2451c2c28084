// shared_attn.cuh -- attention of drafted tokens over a paged cache whose sequences share long prefixes: tree attention's
// kernels over the prefixes, each read once for all rows of its group, and over what the sequences have of their own,
// and the join of the two.
//
// softmax over the union of two sets of keys: with each set's reference m, sum l = sum 2^(z - m) and O = sum 2^(z - m) v,
//   m' = max(m1, m2),  l' = l1 2^(m1 - m') + l2 2^(m2 - m'),  out = (O1 2^(m1 - m') + O2 2^(m2 - m')) / l'.
// Each set's O stays in f32 until this quotient, so that an output is rounded once, as without sharing.
#pragma once

#include "tree_attn.cuh"
#include "tree_attn_fma.cuh"
#include "prefix_tc.cuh"

namespace tgc {

// How a call is cut: both passes as AttnPlan, and the parts of the scratch, in bytes.
struct SharedPlan {
	AttnPlan pre, own;
	int pitch;                 // entries per head of the prefixes' table
	int dp;
	long long least_units;     // of the prefixes: the groups, or their rows if they filled whole tiles
	long long rows;            // seqs * tokens * heads
	size_t tab[2], whole_o[2], whole_ml[2], part[2], bytes; // offsets: prefixes, own positions
};

struct JoinArgs {
	SharedArgs pre, own;
	int pre_rt, own_rt, pre_ctas, own_ctas;
	long long rows;
};

// The parts of a row, prefix first, in the order of their CTAs; a thread has a row and 8 columns. The NG warps of a block
// take the parts in turn, each with a running reference, and the first adds up what they have, in their order: few rows of a long
// prefix have many parts, a chain of loads for one warp.
template <class T, int DP, int NG>
__global__ void __launch_bounds__(32 * (NG > 1 ? NG : 8)) k_shared_join(const JoinArgs p)
{
	__shared__ float s[NG > 1 ? NG : 1][10][32];
	pdl_launch();
	pdl_wait();
	const SharedArgs &a = p.own;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const long long x = NG > 1 ? (long long)blockIdx.x * 32 + lane : (long long)blockIdx.x * 256 + threadIdx.x, row = min(x / (DP / 8), p.rows - 1);
	const int col = (int)(x % (DP / 8)) * 8;
	const bool there = x / (DP / 8) < p.rows;
	const long long bt = quotient(row, (unsigned)a.d.nq);
	const int j = (int)(row - bt * a.d.nq), b = (int)quotient(bt, (unsigned)a.d.tokens), t = (int)(bt - (long long)b * a.d.tokens), h = j / a.d.group, jj = j - h * a.d.group;
	float top = -INFINITY, l = 0, v[8] = {};
	auto add = [&](float m, float n, const float *w) {
		const float to = fmaxf(top, m), f = top == -INFINITY ? 0 : ex2(top - to), g = m == -INFINITY ? 0 : ex2(m - to);
		l = (top == -INFINITY ? l : l * f) + (m == -INFINITY ? n : n * g); // sums keep a NaN
#pragma unroll
		for (int i = 0; i < 8; i++) v[i] = (f == 0 ? 0 : v[i] * f) + (g == 0 ? 0 : w[i] * g);
		top = to;
	};
	// parts k of n: begins at the warp's first, which it leaves for the next list
	int first = NG > 1 ? warp : 0;
	auto parts = [&](const SharedArgs &q, int2 e, int r, int rt, int ctas) {
		const bool whole = e.x == -1;
		// (after a wait that gave up, or with groups that overlap, the entry may be anything)
		if (!whole && (e.x < 0 || e.y < e.x || e.y >= ctas)) return;
		const long long slot = (long long)rt * (DP + 2);
		const int at = rt == 128 ? slot_at<DP, 128>(r, col) : slot_at<DP, 1>(r, col), next = rt == 128 ? 512 : 4;
		const int n = whole ? 1 : e.y - e.x + 1;
#pragma unroll 4
		for (int i = first; i < n; i += NG) {
			const float *o = whole ? q.whole_o + row * DP + col : q.part + (2ll * (e.x + i) + (i == 0)) * slot;
			const float4 y = *(const float4 *)(whole ? o : o + at), z = *(const float4 *)(whole ? o + 4 : o + at + next);
			const float2 ml = whole ? q.whole_ml[row] : make_float2(o[rt * DP + r], o[rt * DP + rt + r]);
			const float w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
			add(ml.x, ml.y, w);
		}
		if (NG > 1) first = (first + NG - n % NG) % NG;
	};
	const int r = t * a.d.group + jj;
	const int2 e = a.tab[((long long)b * a.c.nkv + h) * a.row_tiles + r / p.own_rt];
	int g, n;
	if (a.from(b, n, g) > 0) {
		const int seq = a.first[g], m = a.members[g];
		if (seq < 0 || b < seq || b - seq >= m || m > a.seqs - seq) a.c.report(PG_GROUP);
		const long long r = ((long long)(b - seq) * a.d.tokens + t) * a.d.group + jj, u = p.pre.base(g, seq, p.pre_rt) + r / p.pre_rt;
		if (seq >= 0 && b >= seq && u < p.pre.pitch) parts(p.pre, p.pre.tab[(long long)h * p.pre.pitch + u], (int)(r % p.pre_rt), p.pre_rt, p.pre_ctas);
	}
	parts(a, e, r % p.own_rt, p.own_rt, p.own_ctas);
	if constexpr (NG > 1) {
		if (warp) {
			s[warp][8][lane] = top, s[warp][9][lane] = l;
#pragma unroll
			for (int i = 0; i < 8; i++) s[warp][i][lane] = v[i];
		}
		__syncthreads();
		if (warp) return;
		for (int k = 1; k < NG; k++) {
			float w[8];
#pragma unroll
			for (int i = 0; i < 8; i++) w[i] = s[k][i][lane];
			add(s[k][8][lane], s[k][9][lane], w);
		}
	}
	if (!there) return;
	const AttnRow to = attn_row(a, b, h, r, a.d.drafted(b), l);
	store_row8<T>(a, to, col, v);
	if (col == 0) store_lse(to, top, l);
}

template <int MODE, class T, int DP, int MT>
static int shared_mma(const SharedArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	using A = AttnTile<T, DP, MT>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_tree_attn<T, DP, MT, MODE>;
	int rc = pg_smem(kernel, A::SMEM, pl.dev, done);
	if (rc) return rc;
	TGC_CUDA(launch_pdl(kernel, dim3(pl.grid), dim3(128), A::SMEM, st, p));
	return TG_CUDA_OK;
}

template <int MODE, int DP, int R>
static int shared_fma(const SharedArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	using A = FmaTile<DP, R>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_tree_attn_fma<DP, R, MODE>;
	int rc = pg_smem(kernel, A::SMEM, pl.dev, done);
	if (rc) return rc;
	TGC_CUDA(launch_pdl(kernel, dim3(pl.grid), dim3(128), A::SMEM, st, p));
	return TG_CUDA_OK;
}

template <int MODE, class T, int DP, bool BOX>
static int shared_tc(const SharedArgs &p, const AttnPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	using A = TaTile<DP>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_tree_attn_tc<T, DP, BOX, MODE>;
	if (!(done.load(std::memory_order_acquire) >> pl.dev & 1)) { // see attn_run_tc
		cudaFuncAttributes at;
		TGC_CUDA(cudaFuncGetAttributes(&at, kernel));
		if (at.numRegs < TA_REGS) return set_err(TG_CUDA_EUNSUPPORTED, "shared attention kernel built with %d registers, not %d", at.numRegs, TA_REGS);
	}
	int rc = pg_smem(kernel, A::SMEM, pl.dev, done);
	if (rc) return rc;
	TGC_CUDA(launch_pdl(kernel, dim3(pl.grid), dim3(A::THREADS), A::SMEM, st, p, maps[0], maps[1]));
	return TG_CUDA_OK;
}

template <class T, int DP>
static int prefix_tc(const SharedArgs &p, const AttnPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	using A = PtTile<DP>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_prefix_tc<T, DP>;
	int rc = pg_smem(kernel, A::SMEM, pl.dev, done);
	if (rc) return rc;
	TGC_CUDA(launch_pdl(kernel, dim3(pl.grid), dim3(A::THREADS), A::SMEM, st, p, maps[0], maps[1]));
	return TG_CUDA_OK;
}

// One pass. maps: of the pools, where p.box has rows.
template <int MODE, class T>
static int shared_pass(const SharedArgs &p, const AttnPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	if constexpr (sizeof(T) == 2) {
		if (pl.tc) {
			if constexpr (MODE == ATTN_PREFIX) {
				if (p.box.rows) return pl.dp == 128 ? prefix_tc<T, 128>(p, pl, maps, st) : prefix_tc<T, 64>(p, pl, maps, st);
			} else if (p.box.rows) return pl.dp == 128 ? shared_tc<MODE, T, 128, true>(p, pl, maps, st) : shared_tc<MODE, T, 64, true>(p, pl, maps, st);
			return pl.dp == 128 ? shared_tc<MODE, T, 128, false>(p, pl, maps, st) : shared_tc<MODE, T, 64, false>(p, pl, maps, st);
		}
	}
	if constexpr (sizeof(T) == 4) {
		if (pl.fma == 4) return pl.dp == 256 ? shared_fma<MODE, 256, 4>(p, pl, st) : pl.dp == 128 ? shared_fma<MODE, 128, 4>(p, pl, st) : shared_fma<MODE, 64, 4>(p, pl, st);
		if (pl.fma == 8) return pl.dp == 256 ? shared_fma<MODE, 256, 8>(p, pl, st) : pl.dp == 128 ? shared_fma<MODE, 128, 8>(p, pl, st) : shared_fma<MODE, 64, 8>(p, pl, st);
	}
	if (pl.dp == 256) return shared_mma<MODE, T, 256, 1>(p, pl, st);
	if constexpr (MODE == ATTN_OWN || sizeof(T) == 4) {
		if (pl.dp == 128) return pl.mt == 1 ? shared_mma<MODE, T, 128, 1>(p, pl, st) : shared_mma<MODE, T, 128, 2>(p, pl, st);
		return pl.mt == 1 ? shared_mma<MODE, T, 64, 1>(p, pl, st) : shared_mma<MODE, T, 64, 2>(p, pl, st);
	}
	return set_err(TG_CUDA_EUNSUPPORTED, "shared attention: no kernel"); // (prefixes of 16 bits take the 128-row tiles)
}

// Eight warps a block where the prefixes' units have many parts. The whole call, us, with eight and with one (8 key heads of 128 dimensions, two query
// heads each, bf16): 8 sequences below 2048 positions 18.9 and 21.1, below 16384 31.3 and 44.4; 64 below 2048 39.6 and 40.6; 256 in 8 groups below 8192
// 156 and 151, in 32 groups below 4096 168 and 161; 40 of 21 tokens below 4096 128 and 97; f32: 8 below 4096 34.0 and 39.5.
template <class T, int DP>
static int shared_join(const JoinArgs &j, const SharedPlan &pl, cudaStream_t st)
{
	const long long items = j.rows * (DP / 8);
	if (pl.pre.grid >= 4 * pl.least_units) TGC_CUDA(launch_pdl(k_shared_join<T, DP, 8>, dim3((unsigned)((items + 31) / 32)), dim3(256), 0, st, j));
	else TGC_CUDA(launch_pdl(k_shared_join<T, DP, 1>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, j));
	return TG_CUDA_OK;
}

// The three launches of a planned call; T is the element type.
template <class T>
int shared_type(const JoinArgs &j, const SharedPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	int rc;
	if ((rc = shared_pass<ATTN_PREFIX, T>(j.pre, pl.pre, maps, st)) || (rc = shared_pass<ATTN_OWN, T>(j.own, pl.own, maps, st))) return rc;
	return pl.dp == 256 ? shared_join<T, 256>(j, pl, st) : pl.dp == 128 ? shared_join<T, 128>(j, pl, st) : shared_join<T, 64>(j, pl, st);
}

} // namespace tgc
