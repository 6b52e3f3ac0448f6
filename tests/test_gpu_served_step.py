"""A step of a served batch through the operators together: ternary projections shared by all
requests, each request's adapter beside them, the logits, and each request's next token
under its own settings with its log-probabilities; against 64 bits."""
import numpy as np
import pytest
import torch

from spbitnet_amd import _lib
from spbitnet_amd import kernels as K
from spbitnet_amd import weights as W
from spbitnet_amd.model import InferenceEngine, Model, ModelConfig
from tests import requests64 as R

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, VOCAB = 21, 1024, 4093
SECTIONS = (HIDDEN, 256, 256)


class Projection:
    """A packed ternary layer on the GPU and its dense values on the host."""

    def __init__(self, rows, cols, seed):
        L = W.random_layer(rows, cols, seed)
        self.L, self.rows, self.cols = L, rows, cols
        self.meta = torch.from_numpy(L.meta.view(np.int32)).cuda()
        self.values = torch.from_numpy(L.values.view(np.int32)).cuda()
        self.acc = torch.empty(TOKENS, rows, dtype=torch.int32, device="cuda")

    def run(self, x8, absmax, out):
        """int8 activations through the shared GEMM, dequantised token by token."""
        K.sparse_ternary_gemm_gpu(self.meta, self.values, x8, self.acc, self.rows, self.cols, TOKENS,
                                  self.L.meta_stride, self.L.values_stride)
        for t in range(TOKENS):
            K.dequantize_gpu(self.acc[t], out[t], absmax[t:t + 1], self.L.gamma, self.rows)


def _step(proj, adapters, ids, x, head, uniforms, sampling, buffers):
    """One pass; everything it writes is in buffers."""
    b = buffers
    for t in range(TOKENS):
        K.absmax_reduce_gpu(x[t], b["absmax"][t:t + 1], HIDDEN)
        K.absmax_quantize_gpu(x[t], b["x8"][t], b["absmax"][t:t + 1], HIDDEN)
    proj.run(b["x8"], b["absmax"], b["base"])
    b["out"].copy_(b["base"])
    K.adapters_gpu(adapters, ids, x, b["out"], b["out"], b["adapter_ws"])  # in place
    for t in range(TOKENS):
        _lib.check(_lib.load().spb_gemv_bf16(head.data_ptr(), b["out"][t].data_ptr(), b["logits"][t].data_ptr(),
                                             VOCAB, HIDDEN, torch.cuda.current_stream().cuda_stream or None),
                   "spb_gemv_bf16")
    K.sample_gpu(b["logits"], uniforms, b["tokens"], sampling, b["sample_ws"], logprobs=b["drawn"])
    K.token_logprobs_gpu(b["logits"], b["tokens"], b["logprobs"], b["logprob_ws"], top_ids=b["top_ids"],
                         top_logprobs=b["top_logprobs"])


@pytest.fixture(scope="module")
def served(gpu):
    g = torch.Generator().manual_seed(3)
    rows = sum(SECTIONS)
    proj = Projection(rows, HIDDEN, 11)
    num, rank = 6, 24
    a = (torch.randn(num, 3 * rank, HIDDEN, generator=g) * HIDDEN ** -0.5).bfloat16().cuda()
    b = (torch.randn(num, rows, rank, generator=g) * rank ** -0.5).bfloat16().cuda()
    scales = (torch.rand(num, generator=g) + 0.5).cuda()
    ranks = torch.tensor([24, 8, 1, 16, 24, 5], dtype=torch.int32).cuda()
    adapters = K.Adapters(a, b, scales, ranks=ranks, sections=SECTIONS)
    head = (torch.randn(VOCAB, HIDDEN, generator=g) * 0.05).bfloat16().cuda()
    new = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="cuda")
    buffers = dict(
        absmax=new(TOKENS), x8=new(TOKENS, HIDDEN, dt=torch.int8), base=new(TOKENS, rows, dt=torch.bfloat16),
        out=new(TOKENS, rows, dt=torch.bfloat16), logits=new(TOKENS, VOCAB),
        tokens=new(TOKENS, dt=torch.int32), drawn=new(TOKENS), logprobs=new(TOKENS),
        top_ids=new(TOKENS, 4, dt=torch.int32), top_logprobs=new(TOKENS, 4),
        adapter_ws=new(K.adapters_workspace_size(adapters, TOKENS), dt=torch.uint8),
        sample_ws=new(K.sample_workspace_size(TOKENS, VOCAB), dt=torch.uint8),
        logprob_ws=new(K.token_logprobs_workspace_size(TOKENS, VOCAB, 4), dt=torch.uint8))
    return proj, adapters, head, buffers


def test_step(served):
    proj, adapters, head, buf = served
    g = torch.Generator().manual_seed(8)
    x = torch.randn(TOKENS, HIDDEN, generator=g).bfloat16().cuda()
    ids = torch.randint(-1, 6, (TOKENS,), generator=g, dtype=torch.int32).cuda()
    u = torch.rand(TOKENS, generator=g).cuda()
    t = torch.tensor([(0.0, 0.7, 1.0, 1.3)[i % 4] for i in range(TOKENS)]).cuda()
    k = torch.tensor([(0, 40, 0, 5, 1)[i % 5] for i in range(TOKENS)], dtype=torch.int32).cuda()
    p = torch.tensor([(1.0, 0.9, 0.5)[i % 3] for i in range(TOKENS)]).cuda()
    _step(proj, adapters, ids, x, head, u, K.Sampling(t, k, p, min_p=0.01), buf)
    torch.cuda.synchronize()
    out, err = R.adapters(adapters.a, adapters.b, adapters.scales, adapters.ranks.tolist(), SECTIONS, ids, x,
                          buf["base"])
    assert (np.abs(R.f64(buf["out"]) - out) <= err).all()
    logits = R.f64(buf["logits"])
    u64, t64, p64 = R.f64(u), R.f64(t), R.f64(p)
    for i in range(TOKENS):
        token, lp, _ = R.sample(logits[i], u64[i], t64[i], int(k[i]), p64[i], float(np.float32(0.01)))
        assert int(buf["tokens"][i]) == token, i
        assert abs(float(buf["drawn"][i]) - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -36
        want, bound, best = R.logprobs(logits[i], 4)
        assert abs(float(buf["logprobs"][i]) - want[token]) <= bound[token]
        assert buf["top_ids"][i].tolist() == best.tolist()
        if t64[i] == 0:
            assert token == int(logits[i].argmax()) and lp == 0.0


def test_a_request_is_not_changed_by_its_neighbours(served):
    """Each request alone in the batch (the others without adapter, greedy) answers the same."""
    proj, adapters, head, buf = served
    g = torch.Generator().manual_seed(9)
    x = torch.randn(TOKENS, HIDDEN, generator=g).bfloat16().cuda()
    ids = torch.randint(0, 6, (TOKENS,), generator=g, dtype=torch.int32).cuda()
    u = torch.rand(TOKENS, generator=g).cuda()
    t = torch.full((TOKENS,), 0.8).cuda()
    _step(proj, adapters, ids, x, head, u, K.Sampling(t, top_p=0.9), buf)
    torch.cuda.synchronize()
    tokens, logprobs, out = buf["tokens"].tolist(), buf["logprobs"].tolist(), buf["out"].clone()
    for i in (0, 7, TOKENS - 1):
        alone = torch.full((TOKENS,), -1, dtype=torch.int32).cuda()
        alone[i] = ids[i]
        cold = torch.zeros(TOKENS).cuda()
        cold[i] = 0.8
        _step(proj, adapters, alone, x, head, u, K.Sampling(cold, top_p=0.9), buf)
        torch.cuda.synchronize()
        assert torch.equal(buf["out"][i], out[i])
        assert int(buf["tokens"][i]) == tokens[i] and float(buf["logprobs"][i]) == logprobs[i]


def test_engine_logits_sampled(gpu):
    """The decode engine's logits through sampling, token by token: greedy settings give the
    tokens that generate gives, and drawn tokens are those of the definition."""
    cfg = ModelConfig(hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                      intermediate_size=1536, vocab_size=4096, max_position_embeddings=1024, head_dim=64,
                      rms_norm_eps=1e-5, rope_theta=500000.0, bos_token_id=1, eos_token_id=2)
    eng = InferenceEngine(Model.random(cfg, seed=5), max_seq=256)
    prompt = [7, 300, 21, 4000, 9]
    want = eng.generate(prompt, 6)
    eng.reset()
    for t in prompt[:-1]:
        eng.forward(t)
    ws = torch.empty(K.sample_workspace_size(1, cfg.vocab_size), dtype=torch.uint8, device="cuda")
    token, got, last = torch.empty(1, dtype=torch.int32, device="cuda"), [], prompt[-1]
    u = torch.tensor([0.83], device="cuda")
    for _ in range(len(want)):
        logits = eng.forward(last)[None]
        K.sample_gpu(logits, u, token, K.Sampling(temperature=1.2, top_p=0.7), ws)
        drawn, _, _ = R.sample(R.f64(logits)[0], float(np.float32(0.83)), float(np.float32(1.2)),
                               0, float(np.float32(0.7)))
        assert int(token) == drawn
        K.sample_gpu(logits, u, token, K.Sampling(temperature=0.0), ws)
        last = int(token)
        got.append(last)
    assert got == want
