"""The decoder for several sequences: its attention layer against the formula in 64 bits, and
prompts, single tokens and mixtures of both against the single-sequence decoder."""
import pytest
import torch

from npu_amd import qwen_core as QN, qwen_moe, qwen_serve as QS, synth

pytestmark = pytest.mark.gpu
H = 2.0 ** -8                                            # a rounding to bf16, relative


def _bf(t):
    return t.to(torch.bfloat16).float()


def _attn(cfg, seed):
    g = torch.Generator().manual_seed(seed)
    D, hq, hkv, dh = cfg.d_model, cfg.n_head, cfg.n_head_kv, cfg.head_dim

    def w(*s, sc=0.05):
        return torch.randn(*s, generator=g) * sc
    return QN.AttnLayer(i=0, attn_norm=1 + w(D), post_norm=1 + w(D), wq=_bf(w(2 * hq * dh, D)), wk=_bf(w(hkv * dh, D)),
                        wv=_bf(w(hkv * dh, D)), wo=_bf(w(D, hq * dh)), q_norm=1 + w(dh), k_norm=1 + w(dh))


def _rounded(t):
    """t [n, heads, dim] rounded to bf16, and by how much the rounding of a value within the
    layers' fp32 error (1e-5 of the head's largest) may differ: nothing, or one step."""
    e = 1e-5 * t.abs().amax(-1, keepdim=True)
    r, up, down = (x.to(torch.bfloat16).double() for x in (t, t + e, t - e))
    return r, torch.maximum((up - r).abs(), (down - r).abs())


def _plain(x, L, cfg, steps):
    """The layer on one sequence x [n, D] in 64 bits with k and v rounded to bf16, and q where
    the token came in a step with several (``steps`` True); and a bound on each row's 2-norm of
    the difference: roundings that fall the other way, and for those tokens the softmax
    weights' and the result's rounding."""
    x = x.double()
    n = x.shape[0]
    hq, hkv, dh, half = cfg.n_head, cfg.n_head_kv, cfg.head_dim, cfg.rope_dim // 2
    w = {k: getattr(L, k).double().to(x.device) for k in ("attn_norm", "wq", "wk", "wv", "wo", "q_norm", "k_norm")}

    def norm(t, f):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + cfg.rms_eps) * f
    xn = norm(x, w["attn_norm"])
    q, gate = (xn @ w["wq"].t()).view(n, hq, 2 * dh).split(dh, -1)
    k, v = ((xn @ w[m].t()).view(n, hkv, dh) for m in ("wk", "wv"))
    a = torch.arange(n, device=x.device).double()[:, None] * (
        cfg.rope_theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half))
    c, s = a.cos()[:, None], a.sin()[:, None]

    def turn(t):
        lo, hi = t[..., :half], t[..., half:2 * half]
        return torch.cat([lo * c - hi * s, hi * c + lo * s, t[..., 2 * half:]], -1)
    q, k = turn(norm(q, w["q_norm"])), turn(norm(k, w["k_norm"]))
    many = steps[:, None, None]
    (k, dk), (v, dv), (qr, dq) = _rounded(k), _rounded(v), _rounded(q)
    q, dq = torch.where(many, qr, q), torch.where(many, dq, 1e-5 * q.abs().amax())
    k, v, dk, dv = (t.repeat_interleave(hq // hkv, 1) for t in (k, v, dk, dv))
    live = torch.ones(n, n, dtype=torch.bool, device=x.device).tril()

    def dots(f, g):
        return torch.stack([f[:, h] @ g[:, h].t() for h in range(hq)]) * dh ** -0.5
    p = torch.softmax(dots(q, k).masked_fill(~live, -float("inf")), -1)
    ds = ((dots(q.abs(), dk) + dots(dq, k.abs() + dk)) * live).amax(-1)[..., None]       # how far a score moves
    o, av, sv = (torch.stack([p[h] @ f[:, h] for h in range(hq)]) for f in (v, v.abs(), dv))
    gr = torch.sigmoid(gate).transpose(0, 1)
    r = steps[None, :, None].double() * H                # the weights' rounding, and the result's
    err = ((torch.expm1(2 * ds) + r * torch.exp(2 * ds)) * av + torch.exp(2 * ds) * sv) * gr
    err = err + r * (o.abs() * gr + err)
    y = (o * gr).transpose(0, 1).reshape(n, -1) @ w["wo"].t()
    # through wo by its 2-norm; fp32 sums of the layer as for one sequence
    bound = torch.linalg.matrix_norm(w["wo"], 2) * err.transpose(0, 1).reshape(n, -1).norm(dim=-1)
    return x + y, bound + 1e-4 * (x + y).abs().max() * x.shape[1] ** 0.5


@pytest.mark.parametrize("kw", [dict(n_head=4, n_head_kv=2, head_dim=128, rope_dim=32),
                                dict(n_head=16, n_head_kv=2, head_dim=256, rope_dim=64),
                                dict(n_head=3, n_head_kv=3, head_dim=64, rope_dim=64)])
def test_attention_steps_of_several_sequences(gpu, kw):
    """Prompts of other lengths, single tokens for all, single tokens for some, a prompt beside
    single tokens: every output row against its sequence's formula."""
    print(f"attn_step {kw}", flush=True)
    cfg = QN.Config(d_model=512, n_layer=1, is_attention=[True], rope_theta=1e6, **kw)
    layer = _attn(cfg, 5)
    cache = QS.PagedCache(cfg, 4, 40, page_size=16, dev=gpu)
    rope = QS.build_rope_axes(cfg.rope_dim, cfg.rope_theta)
    plan = [[70, 3, 0, 1], [1, 1, 1, 1], [1, 0, 1, 0], [1, 40, 2, 1], [1, 1, 1, 1], [1, 1, 1, 1]]
    total = [sum(c) for c in zip(*plan)]
    g = torch.Generator(device="cuda").manual_seed(6)
    xs = [torch.randn(n, cfg.d_model, generator=g, device="cuda") for n in total]
    got = [[] for _ in xs]
    many = [[] for _ in xs]
    for counts in plan:
        at = list(cache.length)
        step = cache.reserve(counts)
        x = torch.cat([xs[b][at[b]:at[b] + counts[b]] for b in step.seqs])
        y = QS.attn_step(x, layer, cfg, rope, step, cache.k[0], cache.v[0])
        for b, part in zip(step.seqs, y.split(step.counts)):
            got[b].append(part)
            many[b] += [not step.single] * part.shape[0]
    for b, x in enumerate(xs):
        want, bound = _plain(x, layer, cfg, torch.tensor(many[b], device="cuda"))
        out = torch.cat(got[b]).double()
        off = (out - want).norm(dim=-1)
        assert bool((off <= bound).all()), (b, float((off / bound).max()))
        # the bound is far below what the layer adds, so that a wrong row or position shows
        assert float(bound.median()) < 0.25 * float((want - x.double()).norm(dim=-1).median())


def _model(seed, n_layer=4):
    cfg = QN.Config(d_model=512, n_layer=n_layer, n_head=4, n_head_kv=2, head_dim=128, rope_dim=32, rope_theta=1e6,
                    ssm_d_inner=256, ssm_d_state=64, ssm_n_k_heads=2, ssm_n_v_heads=4, n_expert=16, n_expert_used=4,
                    d_expert_ff=256, is_attention=[(i + 1) % 2 == 0 for i in range(n_layer)])
    g = torch.Generator().manual_seed(seed)

    def w(*s, sc=0.02):
        return torch.randn(*s, generator=g) * sc
    cores = []
    for i in range(n_layer):
        if cfg.is_attention[i]:
            cores.append(_attn(cfg, seed + i))
        else:
            D, Hv, Hk, S = cfg.d_model, cfg.ssm_n_v_heads, cfg.ssm_n_k_heads, cfg.ssm_d_state
            C = 2 * Hk * S + Hv * S
            cores.append(QN.SSMLayer(i=i, attn_norm=1 + w(D), post_norm=1 + w(D), w_in=_bf(w(C, D)),
                                     w_gate=_bf(w(Hv * S, D)), conv1d=w(C, cfg.ssm_d_conv, sc=0.5),
                                     a=-torch.rand(Hv, generator=g) * 2, alpha=w(Hv, D), beta=w(Hv, D),
                                     dt_bias=w(Hv), ssm_norm=1 + w(S), w_out=_bf(w(D, Hv * S))))
    hs = [synth.host_moe_layer(seed + i, D=512, FF=256, E=16, k=4) for i in range(n_layer)]
    ts = qwen_moe.SyntheticTensorStore(hs)
    cos, sin = QN.build_partial_rope_cache(cfg.rope_dim, 128, cfg.rope_theta)
    return QN.Model(cfg=cfg, token_embd=torch.randn(1000, 512, generator=g), output_norm=1 + w(512),
                    lm_head=_bf(w(1000, 512, sc=0.05)), rope_cos=cos, rope_sin=sin,
                    layers=[(cores[i], qwen_moe.MoELayer.load(ts, i)) for i in range(n_layer)])


def test_decoder_steps_against_one_sequence_each(gpu):
    """Logits of mixed steps beside ``qwen_core.forward`` on each sequence alone, without the
    MoE blocks (whose router may choose other experts for a rounding's difference).  Two
    attention layers round k, v, q, weights and result to bf16, ten roundings of 2^-8, so the
    bar is 4% of the largest logit; a row or position mixed up changes all of it."""
    model = _model(50)
    cfg = model.cfg
    cache = QS.PagedCache(cfg, 3, 12, dev=gpu)
    g = torch.Generator().manual_seed(8)
    plan = [[33, 5, 0], [1, 1, 0], [1, 1, 17], [1, 1, 1], [0, 3, 1]]
    seqs = [torch.randint(0, 1000, (sum(c),), generator=g).tolist() for c in zip(*plan)]
    alone = [QN.forward(model, s, skip_moe=True)[0] for s in seqs]
    for counts in plan:
        at = list(cache.length)
        logits = QS.forward_step(model, [s[a:a + n] for s, a, n in zip(seqs, at, counts)], cache, skip_moe=True)
        assert logits.shape == (sum(n > 0 for n in counts), 1000)
        for row, b in zip(logits, [b for b in range(3) if counts[b]]):
            want = alone[b][cache.length[b] - 1]
            assert float((row - want).abs().max()) <= 10 * H * float(want.abs().max()), (counts, b)
    assert QS.forward_step(model, [[], [], []], cache).shape == (0, 1000)
    with pytest.raises(ValueError, match="tokens must be"):
        QS.forward_step(model, [[1000], [], []], cache)


def test_generation(gpu):
    """Greedy tokens are the argmax of the steps' logits with the MoE blocks in, a drawn run
    repeats with its generator, ``stop`` ends a sequence, and the pages all come back."""
    model = _model(90)
    prompts = [[3, 141, 59], [26], [535, 897, 93, 238, 462, 643, 383, 279]]
    cache = QS.PagedCache(model.cfg, 3, 9, page_size=8, dev=gpu)
    out = QS.generate(model, prompts, 6, cache, temperature=0.0)
    assert [len(o) for o in out] == [6, 6, 6] and sorted(cache.free) == list(range(9)) and cache.length == [0, 0, 0]
    new = prompts
    for i in range(6):
        logits = QS.forward_step(model, new, cache)
        assert logits.argmax(-1).tolist() == [o[i] for o in out]
        new = [[o[i]] for o in out]
    for b in range(3):
        cache.release(b)
    runs = [QS.generate(model, prompts, 5, cache, temperature=0.8, top_k=50, top_p=0.9, min_p=0.01,
                        generator=torch.Generator(device="cuda").manual_seed(3)) for _ in range(2)]
    assert runs[0] == runs[1] and all(0 <= t < 1000 for o in runs[0] for t in o)
    stop = out[1][2]
    ended = QS.generate(model, prompts, 6, cache, temperature=0.0, stop=stop)
    for full, o in zip(out, ended):
        n = full.index(stop) + 1 if stop in full else 6
        assert len(o) == n and o[0] == full[0]
    with pytest.raises(MemoryError):
        QS.generate(model, prompts, 60, cache, temperature=0.0)
    assert sorted(cache.free) == list(range(9))
