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
#include "tree_attn_tc.cuh"

namespace tgc {

// How a call is cut: both passes as AttnPlan, and the parts of the scratch, in bytes.
struct SharedPlan {
	AttnPlan pre, own;
	int pitch;                 // entries per head of the prefixes' table
	int dp;
	long long rows;            // seqs * tokens * heads
	size_t tab[2], whole_o[2], whole_ml[2], part[2], bytes; // offsets: prefixes, own positions
};

struct JoinArgs {
	SharedArgs pre, own;
	int pre_rt, own_rt, pre_ctas, own_ctas;
	long long rows;
};

// The parts of a row, a thread for 8 columns, in the order of their CTAs: prefix first.
template <class T, int DP>
__global__ void __launch_bounds__(256) k_shared_join(const JoinArgs p)
{
	pdl_launch();
	pdl_wait();
	const SharedArgs &a = p.own;
	const long long x = (long long)blockIdx.x * 256 + threadIdx.x, row = x / (DP / 8);
	const int col = (int)(x % (DP / 8)) * 8;
	if (row >= p.rows) return;
	const long long bt = row / a.d.nq;
	const int j = (int)(row - bt * a.d.nq), b = (int)(bt / a.d.tokens), t = (int)(bt - (long long)b * a.d.tokens), h = j / a.d.group, jj = j - h * a.d.group;
	float top = -INFINITY, l = 0, v[8] = {};
	auto add = [&](float m, float n, float4 y, float4 z) {
		const float w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
		const float to = fmaxf(top, m), f = top == -INFINITY ? 0 : ex2(top - to), g = m == -INFINITY ? 0 : ex2(m - to);
		l = (top == -INFINITY ? l : l * f) + (m == -INFINITY ? n : n * g); // sums keep a NaN
#pragma unroll
		for (int i = 0; i < 8; i++) v[i] = (f == 0 ? 0 : v[i] * f) + (g == 0 ? 0 : w[i] * g);
		top = to;
	};
	auto parts = [&](const SharedArgs &s, int2 e, int r, int rt, int ctas) {
		if (e.x == -1) {
			const float *o = s.whole_o + row * DP + col;
			const float2 ml = s.whole_ml[row];
			add(ml.x, ml.y, *(const float4 *)o, *(const float4 *)(o + 4));
			return;
		}
		// (after a wait that gave up, or with groups that overlap, the entry may be anything)
		if (e.x < 0 || e.y < e.x || e.y >= ctas) return;
		const long long slot = (long long)rt * (DP + 2);
		const int at = rt == 128 ? slot_at<DP, 128>(r, col) : slot_at<DP, 1>(r, col), next = rt == 128 ? 512 : 4;
#pragma unroll 4
		for (int i = e.x; i <= e.y; i++) {
			const float *q = s.part + (2ll * i + (i == e.x)) * slot;
			add(q[rt * DP + r], q[rt * DP + rt + r], *(const float4 *)(q + at), *(const float4 *)(q + at + next));
		}
	};
	int g, seq, m, n;
	const int from = a.from(b, a.c.length(b), g);
	if (g >= 0 && from > 0) {
		p.pre.prefix(g, seq, m, n);
		if (n > 0 && b >= seq && b - seq < m) {
			const long long r = ((long long)(b - seq) * a.d.tokens + t) * a.d.group + jj, u = p.pre.base(g, seq, p.pre_rt) + r / p.pre_rt;
			if (u < p.pre.pitch) parts(p.pre, p.pre.tab[(long long)h * p.pre.pitch + u], (int)(r % p.pre_rt), p.pre_rt, p.pre_ctas);
		}
	}
	const int r = t * a.d.group + jj;
	parts(a, a.tab[((long long)b * a.c.nkv + h) * a.row_tiles + r / p.own_rt], r % p.own_rt, p.own_rt, p.own_ctas);
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

template <int DP, int R>
static int shared_fma(const SharedArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	using A = FmaTile<DP, R>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_tree_attn_fma<DP, R, ATTN_OWN>;
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

// One pass. maps: of the pools, where p.box has rows.
template <int MODE, class T>
static int shared_pass(const SharedArgs &p, const AttnPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	if constexpr (sizeof(T) == 2) {
		if (pl.tc) {
			if (p.box.rows) return pl.dp == 128 ? shared_tc<MODE, T, 128, true>(p, pl, maps, st) : shared_tc<MODE, T, 64, true>(p, pl, maps, st);
			return pl.dp == 128 ? shared_tc<MODE, T, 128, false>(p, pl, maps, st) : shared_tc<MODE, T, 64, false>(p, pl, maps, st);
		}
	}
	if constexpr (MODE == ATTN_OWN && sizeof(T) == 4) {
		if (pl.fma == 4) return pl.dp == 256 ? shared_fma<256, 4>(p, pl, st) : pl.dp == 128 ? shared_fma<128, 4>(p, pl, st) : shared_fma<64, 4>(p, pl, st);
		if (pl.fma == 8) return pl.dp == 256 ? shared_fma<256, 8>(p, pl, st) : pl.dp == 128 ? shared_fma<128, 8>(p, pl, st) : shared_fma<64, 8>(p, pl, st);
	}
	if (pl.dp == 256) return shared_mma<MODE, T, 256, 1>(p, pl, st);
	if constexpr (MODE == ATTN_OWN || sizeof(T) == 4) {
		if (pl.dp == 128) return pl.mt == 1 ? shared_mma<MODE, T, 128, 1>(p, pl, st) : shared_mma<MODE, T, 128, 2>(p, pl, st);
		return pl.mt == 1 ? shared_mma<MODE, T, 64, 1>(p, pl, st) : shared_mma<MODE, T, 64, 2>(p, pl, st);
	}
	return set_err(TG_CUDA_EUNSUPPORTED, "shared attention: no kernel"); // (prefixes of 16 bits take the 128-row tiles)
}

template <class T, int DP>
static int shared_join(const JoinArgs &j, cudaStream_t st)
{
	TGC_CUDA(launch_pdl(k_shared_join<T, DP>, dim3((unsigned)((j.rows * (DP / 8) + 255) / 256)), dim3(256), 0, st, j));
	return TG_CUDA_OK;
}

// The three launches of a planned call; T is the element type.
template <class T>
int shared_type(const JoinArgs &j, const SharedPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	int rc;
	if ((rc = shared_pass<ATTN_PREFIX, T>(j.pre, pl.pre, maps, st)) || (rc = shared_pass<ATTN_OWN, T>(j.own, pl.own, maps, st))) return rc;
	return pl.dp == 256 ? shared_join<T, 256>(j, st) : pl.dp == 128 ? shared_join<T, 128>(j, st) : shared_join<T, 64>(j, st);
}

} // namespace tgc
