"""The serving operators where the model uses them: 8-bit MLPs and head, and drawn tokens, in prompts, cached steps and graphs."""
import copy

import pytest
import torch
from torch import nn

import solvedelta_b200 as sd
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def _model(seed=0, hidden=256, heads=4, layers=2, vocab=1000, **more):
    torch.manual_seed(seed)
    config = sd.SolveDeltaConfig(hidden_size=hidden, num_heads=heads, num_hidden_layers=layers, vocab_size=vocab, initializer_range=0.05, **more)
    return sd.SolveDeltaForCausalLM(config).prepare("cuda").eval()


def _ids(model, batch, length, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, model.vocab_size, (batch, length), generator=gen, device="cuda")


@pytest.mark.parametrize("rows", (1, 7, 40, 300))
@pytest.mark.parametrize("width,inner,bias", ((256, 512, False), (1024, 2816, False), (200, 88, True)))
def test_gated_mlp_is_its_two_projections(rows, width, inner, bias):
    """One native call, whose second product is chained to the first: the same bits, again and again."""
    torch.manual_seed(rows + width)
    x = torch.randn(rows, width, device="cuda").to(torch.bfloat16)
    up, up_scale = sd.quantize_rows(torch.randn(2 * inner, width, device="cuda") / width ** 0.5)
    down, down_scale = sd.quantize_rows(torch.randn(width, inner, device="cuda") / inner ** 0.5)
    b = torch.randn(2 * inner, device="cuda") if bias else None
    act = sd.int8_linear(x, up, up_scale, b, swiglu=True)
    want = sd.int8_linear(act, down, down_scale)
    torch.cuda.synchronize()
    for _ in range(20):
        assert torch.equal(sd.int8_gated_mlp(x, up, up_scale, b, down, down_scale, None), want)
    q, scale = ref.quantize(ref.as64(act))
    exact, size = ref.projection(q, scale, ref.as64(down), ref.as64(down_scale))
    exact, bound = ref.projection_bound(exact, size, 2.0 ** -7, False)
    assert (abs(ref.as64(want) - exact) <= bound).all()


def test_int8_linear_module():
    for width, columns, bias in ((256, 96, True), (100, 33, True), (77, 10, False)):
        linear = nn.Linear(width, columns, bias=bias).to("cuda", torch.bfloat16)
        made = sd.Int8Linear.from_linear(linear)
        x = torch.randn(3, 5, width, device="cuda").to(torch.bfloat16)
        q, scale = sd.quantize_rows(linear.weight)
        with torch.no_grad():
            want = sd.int8_linear(x, q, scale, linear.bias)
            assert torch.equal(made(x), want)
            twin = sd.Int8Linear(width, columns, bias=bias)
            twin.load_state_dict({k: v.cpu() for k, v in made.state_dict().items()})
            for other in (twin.cuda(), copy.deepcopy(made), copy.deepcopy(made).bfloat16(), copy.deepcopy(made).half(), made.cpu().cuda()):
                assert other.weight.stride(0) % 16 == 0 and other.weight_scale.dtype == torch.float32
                assert torch.equal(other(x), want)
        assert not list(made.parameters())
        with pytest.raises(RuntimeError, match="no reverse pass"):
            made(x.requires_grad_())
    broken = nn.Linear(16, 16, device="cuda")
    with torch.no_grad():
        broken.weight[3, 3] = float("nan")
    with pytest.raises(ValueError, match="cannot be quantised"):
        sd.Int8Linear.from_linear(broken)


@pytest.mark.parametrize("head", (False, True))
def test_quantized_model(head):
    """Prompt, cached tokens and graph of a quantised model, against its own modules and near the BF16 model.

    Rounding to 8 bits is off by a / 127 / sqrt(12) on average, a the largest magnitude of a row: for 256 normal entries (a
    about 3.5 deviations, at most 6) 0.8 to 1.4 percent, for weights as much, for the activation between the two products
    (a up to 20 deviations) 5 percent; one MLP adds in squares to less than 6 percent of its own output, a layer's output
    holds that and the mixer's, and the head adds 2: less than 10 percent of the logits."""
    model = _model()
    ids = _ids(model, 3, 40)
    with torch.no_grad():
        plain = model(input_ids=ids).logits.float()
        model.quantize_int8(head=head)
        assert isinstance(model.model.layers[0].mlp.up_proj if hasattr(model.model.layers[0].mlp, "up_proj") else
                          model.model.layers[0].mlp.gate_up_proj, sd.Int8Linear)
        assert isinstance(model.lm_head, sd.Int8Linear) == head
        again = model.quantize_int8(head=head)
        assert again is model
        out = model(input_ids=ids, use_cache=True)
        logits = out.logits.float()
        off = (logits - plain).norm() / plain.norm()
        assert 1e-4 < off.item() < 0.1
        mlp = model.model.layers[0].mlp
        x = torch.randn(5, 256, device="cuda").to(torch.bfloat16)
        act = sd.int8_linear(x, mlp.gate_up_proj.weight, mlp.gate_up_proj.weight_scale, swiglu=True)
        assert torch.equal(mlp(x), mlp.down_proj(act))
    assert torch.equal(model.greedy_generate(ids, 6), model.greedy_generate(ids, 6, graphed=True))
    with pytest.raises(RuntimeError, match="no reverse pass"):
        model(input_ids=ids)   # gradients recorded


def test_a_quantised_mlp_with_hooks_runs_its_modules():
    model = _model(layers=1).quantize_int8()
    mlp, seen = model.model.layers[0].mlp, []
    x = torch.randn(2, 256, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        want = mlp(x)
        handle = mlp.gate_up_proj.register_forward_hook(lambda module, args, out: seen.append(out.shape[-1]))
        got = mlp(x)
        handle.remove()
    assert seen == [mlp.gate_up_proj.out_features]
    # the separate product rounds gate and value to BF16 before the activation: a step of 2^-8 of each, through two products
    assert ((got - want).float().norm() / want.float().norm()).item() < 2e-2


def test_quantising_a_model_that_has_decoded():
    """The native stack of the BF16 layers does not outlive them: the same bits as a model that was quantised first."""
    model = _model()
    first = copy.deepcopy(model).quantize_int8()
    ids = _ids(model, 2, 9)
    model.greedy_generate(ids, 3)
    model.quantize_int8()
    with torch.no_grad():
        logits = []
        for m in (first, model):
            step = m(input_ids=ids, use_cache=True)
            logits.append([step.logits])
            for n in range(3):
                step = m(input_ids=ids[:, n:n + 1], past_key_values=step.past_key_values, use_cache=True)
                logits[-1].append(step.logits)
    assert all(torch.equal(a, b) for a, b in zip(*logits))


def test_tied_heads_are_refused():
    with pytest.raises(ValueError, match="tied head"):
        _model(tie_word_embeddings=True).quantize_int8(head=True)


@pytest.mark.parametrize("quantised", (False, True))
def test_drawn_tokens(quantised):
    """Every token is the definition's for the logits of the step before it; graphed and not."""
    model = _model(seed=3)
    if quantised:
        model.quantize_int8(head=True)
    ids = _ids(model, 4, 17)
    settings = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.5], device="cuda"), top_k=torch.tensor([0, 20, 0, 3], dtype=torch.int32, device="cuda"),
                    top_p=0.95, min_p=torch.tensor([0.0, 0.0, 0.05, 0.0], device="cuda"))
    uniform = torch.rand(5, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    got = model.sample_generate(ids, 5, uniform=uniform, **settings)
    assert got.shape == (4, 22) and torch.equal(got[:, :17], ids)
    assert torch.equal(got, model.sample_generate(ids, 5, uniform=uniform, graphed=True, **settings))
    assert torch.equal(got[0], model.greedy_generate(ids, 5)[0])
    with torch.no_grad():
        step = model(input_ids=ids, use_cache=True, logits_to_keep=1)
        for n in range(5):
            want = ref.tokens(step.logits[:, -1], uniform[n], **{k: v for k, v in settings.items()})
            assert got[:, 17 + n].tolist() == want
            step = model(input_ids=got[:, 17 + n:18 + n], past_key_values=step.past_key_values, use_cache=True)


def test_draws_follow_the_generator():
    model = _model(layers=1)
    ids = _ids(model, 2, 5)

    def run(seed):
        return model.sample_generate(ids, 8, temperature=1.2, generator=torch.Generator(device="cuda").manual_seed(seed))

    assert torch.equal(run(1), run(1)) and not torch.equal(run(1), run(2))
    with pytest.raises(ValueError, match="max_new_tokens, B"):
        model.sample_generate(ids, 8, uniform=torch.rand(8, 3, device="cuda"))
    assert torch.equal(model.sample_generate(ids, 0), ids)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_a_module_keeps_the_type_of_its_bias(dtype):
    torch.manual_seed(4)
    linear = nn.Linear(96, 40, device="cuda", dtype=dtype)
    with torch.no_grad():
        linear.bias.copy_(torch.randn(40) + 1 / 3)
    made = sd.Int8Linear.from_linear(linear)
    assert made.bias.dtype == dtype and torch.equal(made.bias, linear.bias.detach())
    x = torch.randn(5, 96, device="cuda").to(torch.bfloat16)
    q, scale = sd.quantize_rows(linear.weight.detach())
    assert torch.equal(made(x), sd.int8_linear(x, q, scale, linear.bias.detach()))
    twin = sd.Int8Linear(96, 40, bias=True, device="cuda", bias_dtype=dtype)
    twin.load_state_dict(made.state_dict())
    assert torch.equal(twin(x), made(x))
    assert copy.deepcopy(made).bfloat16().bias.dtype == torch.bfloat16 and copy.deepcopy(made).half().bias.dtype == torch.bfloat16


@pytest.mark.parametrize("fused", (dict(fuse_linear_cross_entropy=True, fuse_cross_entropy=False), dict(fuse_cross_entropy=True),
                                   dict(fuse_cross_entropy=False)))
def test_loss_of_a_quantised_head(fused):
    """The loss is that of the logits which the head gives, whichever way the configuration computes losses."""
    model = _model(layers=1, **fused).quantize_int8(head=True)
    ids = _ids(model, 2, 21)
    labels = ids.clone()
    labels[0, 4:9] = -100
    with torch.no_grad():
        loss = model(input_ids=ids, labels=labels).loss
        logits = model(input_ids=ids).logits.double()
    want = nn.functional.cross_entropy(logits[:, :-1].reshape(-1, 1000), labels[:, 1:].reshape(-1))
    # FP32: a sum of 1000 exponentials is 1000 * 2^-24 of itself off at most, so its logarithm is 6e-5 off; the loss is near log 1000
    assert abs(loss.item() - want.item()) <= 1e-4 * want.item()
    if fused.get("fuse_linear_cross_entropy"):   # nothing counted: 0, as with a head in BF16
        with torch.no_grad():
            assert model(input_ids=ids, labels=torch.full_like(ids, -100)).loss.item() == 0.0
    with torch.no_grad(), pytest.raises(TypeError, match="weight must be"):
        sd.causal_lm_loss(model, ids, labels, total=35)


@pytest.mark.parametrize("hidden,heads", ((128, 2), (192, 2), (320, 4)))
@pytest.mark.parametrize("rows", (1, 16))
def test_quantised_models_of_odd_widths_decode(hidden, heads, rows):
    """Widths that are no whole groups of 256: a cached token against the last of the whole prompt.  The two round differently
    in BF16, so entries next to a half go to the other integer; that is less than all of the quantisation, 10 percent (see above)."""
    model = _model(hidden=hidden, heads=heads, vocab=300).quantize_int8()
    ids = _ids(model, rows, 12)
    with torch.no_grad():
        step = model(input_ids=ids, use_cache=True)
        whole = model(input_ids=torch.cat((ids, ids[:, :1]), dim=1)).logits[:, -1].float()
        got = model(input_ids=ids[:, :1], past_key_values=step.past_key_values, use_cache=True).logits[:, -1].float()
    assert torch.isfinite(got).all() and ((got - whole).norm() / whole.norm()).item() < 0.1


def test_a_model_is_quantised_as_a_whole_or_not_at_all():
    model = _model()
    last = model.model.layers[-1].mlp.down_proj
    handle = last.register_forward_hook(lambda module, args, out: 2 * out)
    with pytest.raises(TypeError, match="plain nn.Linear"):
        model.quantize_int8(head=True)
    assert not any(isinstance(module, sd.Int8Linear) for module in model.modules())
    handle.remove()
    model.quantize_int8()
    assert sum(isinstance(module, sd.Int8Linear) for module in model.modules()) == 4
    assert type(model.lm_head) is nn.Linear
    kept = model.model.layers[0].mlp.gate_up_proj
    model.quantize_int8(head=True)
    assert isinstance(model.lm_head, sd.Int8Linear) and model.model.layers[0].mlp.gate_up_proj is kept
