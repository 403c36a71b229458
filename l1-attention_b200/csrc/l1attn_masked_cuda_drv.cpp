// pybind module l1attn_masked_cuda_drv: masked L1 attention on torch tensors -- checks, allocation, device and stream; the
// arithmetic is behind the C ABI (l1attn_masked_fwd / _bwd).
#include <c10/util/Optional.h>
#include "drv_common.h"

namespace {

using Maybe = c10::optional<torch::Tensor>;

const char *const SHAPES = "q must be [bs, n, h, w], k [bs, n, hk, w], v [bs, n, hk, wv]";

// a small tensor beside q, k, v: its shape, type and device; contiguous.  record: gradients are wanted
torch::Tensor side(const Maybe &t, const char *name, at::IntArrayRef shape, torch::ScalarType type, const torch::Tensor &like, bool record)
{
	if (!t.has_value() || !t->defined())
		return {};
	TORCH_CHECK(t->scalar_type() == type && t->sizes() == shape && t->device() == like.device(), name, " must be a ", type, " tensor of shape ", l1b_shape(shape),
		    " on the device of q");
	TORCH_CHECK(!(record && t->requires_grad()), name, " is a constant: it must not require a gradient");
	l1b_no_tangent(*t, name);
	return t->contiguous();
}

torch::Tensor rows(const torch::Tensor &t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }

struct Call {
	torch::Tensor q, k, v, slopes, doc, prefix;
	l1attn_mask mask;
	int64_t strides[9];
	int bs, n, h, hk, w, wv, type;

	Call(const torch::Tensor &q_, const torch::Tensor &k_, const torch::Tensor &v_, const Maybe &slopes_, const Maybe &doc_, const Maybe &prefix_, int mode, bool causal,
	     int64_t window, double softcap, bool record)
	{
		CHECK_CUDA(q_);
		CHECK_CUDA(k_);
		CHECK_CUDA(v_);
		TORCH_CHECK(q_.dim() == 4 && k_.dim() == 4 && v_.dim() == 4, SHAPES);
		TORCH_CHECK(k_.size(0) == q_.size(0) && k_.size(1) == q_.size(1) && k_.size(3) == q_.size(3) && v_.sizes().slice(0, 3) == k_.sizes().slice(0, 3), SHAPES);
		TORCH_CHECK(k_.size(2) ? q_.size(2) > 0 && q_.size(2) % k_.size(2) == 0 : q_.size(2) == 0, "the heads of q must be a multiple of those of k and v");
		const auto t = q_.scalar_type();
		TORCH_CHECK((t == torch::kFloat32 || t == torch::kFloat16 || t == torch::kBFloat16) && k_.scalar_type() == t && v_.scalar_type() == t,
			    "q, k, v must share dtype float32, float16 or bfloat16");
		TORCH_CHECK(k_.device() == q_.device() && v_.device() == q_.device(), "q, k, v must be on one device");
		TORCH_CHECK(q_.size(3) >= 1 && q_.size(3) <= 256 && v_.size(3) >= 1 && v_.size(3) <= 256, "widths must be 1 to 256");
		for (int64_t s : {q_.size(0), q_.size(1), q_.size(2)})
			TORCH_CHECK(s <= 1 << 30, "sizes must be 2^30 at most");
		l1b_no_tangent(q_, "q");
		l1b_no_tangent(k_, "k");
		l1b_no_tangent(v_, "v");
		q = rows(q_);
		k = rows(k_);
		v = rows(v_);
		slopes = side(slopes_, "slopes", {q.size(2)}, torch::kFloat32, q, record);
		doc = side(doc_, "doc", {q.size(0), q.size(1)}, torch::kInt32, q, record);
		prefix = side(prefix_, "prefix", {q.size(0)}, torch::kInt32, q, record);
		const torch::Tensor *const all[] = {&q, &k, &v};
		for (int i = 0; i < 9; i++)
			strides[i] = all[i / 3]->stride(i % 3);
		bs = int(q.size(0));
		n = int(q.size(1));
		h = int(q.size(2));
		hk = int(k.size(2));
		w = int(q.size(3));
		wv = int(v.size(3));
		type = l1b_dtype(q, "masked attention", true);
		mask = {causal, int(window), mode, float(softcap), slopes.defined() ? slopes.data_ptr<float>() : nullptr, doc.defined() ? doc.data_ptr<int32_t>() : nullptr,
			prefix.defined() ? prefix.data_ptr<int32_t>() : nullptr};
	}
	torch::Tensor work(int backward) const
	{
		if (!backward && !doc.defined())
			return {};
		return torch::empty({int64_t(l1attn_masked_work_bytes(bs, n, h, hk, w, wv, type, backward))}, q.options().dtype(torch::kUInt8).requires_grad(false));
	}
};

void *ptr(const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// -> [vo], or (keep) [vo, rest, lse] -- rest: what rounding to 16 bits left of vo, undefined in float32 -- and what the backward takes: q, k, v, slopes, doc, prefix as they were used
std::vector<torch::Tensor> forward(torch::Tensor q, torch::Tensor k, torch::Tensor v, Maybe slopes, Maybe doc, Maybe prefix, int mode, bool causal, int64_t window,
				   double softcap, bool keep)
{
	const Call c(q, k, v, slopes, doc, prefix, mode, causal, window, softcap, keep || at::GradMode::is_enabled());
	const c10::cuda::CUDAGuard guard(c.q.device());
	const auto options = c.q.options().requires_grad(false);
	auto vo = torch::empty({c.bs, c.n, c.h, c.wv}, options);
	torch::Tensor lse = keep ? torch::empty({c.bs, c.n, c.h}, options.dtype(torch::kFloat32)) : torch::Tensor();
	torch::Tensor rest = keep && c.type != L1ATTN_F32 ? torch::empty_like(vo) : torch::Tensor();
	const auto work = c.work(0);
	l1b_status(l1attn_masked_fwd(ptr(c.q), ptr(c.k), ptr(c.v), c.strides, ptr(vo), ptr(rest), static_cast<float *>(ptr(lse)), ptr(work), c.bs, c.n, c.h, c.hk, c.w, c.wv, &c.mask, c.type,
				     l1b_stream()),
		   "l1attn_masked_fwd");
	if (!keep)
		return {vo};
	return {vo, rest, lse, c.q, c.k, c.v, c.slopes, c.doc, c.prefix};
}

std::vector<torch::Tensor> backward(torch::Tensor q, torch::Tensor k, torch::Tensor v, Maybe slopes, Maybe doc, Maybe prefix, int mode, bool causal, int64_t window,
				    double softcap, torch::Tensor vo, Maybe rest, torch::Tensor lse, torch::Tensor dvo)
{
	const Call c(q, k, v, slopes, doc, prefix, mode, causal, window, softcap, false);
	TORCH_CHECK(dvo.sizes() == vo.sizes() && dvo.scalar_type() == vo.scalar_type() && dvo.device() == vo.device(), "the gradient must be like the output");
	const c10::cuda::CUDAGuard guard(c.q.device());
	dvo = dvo.contiguous();
	const auto options = c.q.options().requires_grad(false);
	auto dq = torch::empty(c.q.sizes(), options), dk = torch::empty(c.k.sizes(), options), dv = torch::empty(c.v.sizes(), options);
	const auto work = c.work(1);
	l1b_status(l1attn_masked_bwd(ptr(c.q), ptr(c.k), ptr(c.v), c.strides, ptr(vo), rest.has_value() ? ptr(*rest) : nullptr, ptr(dvo), lse.data_ptr<float>(), ptr(dq), ptr(dk), ptr(dv), ptr(work), c.bs, c.n, c.h, c.hk,
				     c.w, c.wv, &c.mask, c.type, l1b_stream()),
		   "l1attn_masked_bwd");
	return {dq, dk, dv};
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
	m.def("forward", &forward, "masked L1 attention (CUDA, sm_100a)");
	m.def("backward", &backward, "gradients of masked L1 attention (CUDA, sm_100a)");
}
