"""GPU: the decode loop with the attention mixer in its layers -- the library's paged cache and attention against plain PyTorch
ops over the values read back from the same kind of cache."""

import pytest
import torch

from fastkernels_b200.spec import MoESpec, synthetic_qwen36_spec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_both_impls_agree_on_a_four_layer_tiny_model(cache_dtype, window, sinks):
    from fastkernels_b200.decode_runner import DecodeRunner, build_layers
    spec = synthetic_qwen36_spec()
    layers = build_layers(spec, 4, torch.float32, "cuda")
    outs = {}
    for impl in ("reference", "b200"):
        runner = DecodeRunner(layers, spec, moe_impl=impl, dtype=torch.float32, seed=3, vocab=64, mixer="attention", max_positions=64, cache_dtype=cache_dtype,
                              window=window, sinks=sinks)
        first = runner.generate([1, 7, 3], 12)
        runner.reset()
        generated, logits = runner.generate([1, 7, 3], 12)
        assert generated == first[0] and torch.equal(logits, first[1])          # a reset cache starts anew
        assert runner.mixers[0].cache.host_lengths == [15]
        outs[impl] = (generated, logits.clone())
    assert outs["reference"][0] == outs["b200"][0]
    # fp32 throughout; with an 8-bit cache a rounding of 2^-24 before the quantiser can move a code (a step of 2^-3 of a value) in one arm
    atol = 1e-4 if cache_dtype is None else 2e-2
    torch.testing.assert_close(outs["b200"][1], outs["reference"][1], atol=atol, rtol=1e-4)


def test_real_shape_two_layers_bf16():
    from fastkernels_b200.decode_runner import DecodeRunner, build_layers
    spec = MoESpec()
    layers = build_layers(spec, 2, torch.bfloat16, "cuda")
    logits = {}
    for impl in ("reference", "b200"):
        runner = DecodeRunner(layers, spec, moe_impl=impl, dtype=torch.bfloat16, seed=4, vocab=128, mixer="attention", max_positions=32)
        for token in (5, 9, 5, 77):
            out = runner.step(token)
        logits[impl] = out.clone()
    # the residual stream passes through bf16 before each sublayer in both arms (2^-8 of a value of order 1, twice per layer), the
    # logits sum 2048 of them with weights of 0.02: sqrt(2048) * 0.02 * 2^-8 * 4 = 1.4e-2
    torch.testing.assert_close(logits["b200"], logits["reference"], atol=2e-2, rtol=2e-2)


def test_cli_names_the_mixer(capsys):
    from fastkernels_b200 import decode_runner
    decode_runner.main(["--spec", "tiny", "--dtype", "float32", "--layers", "2", "--prompt-token-ids", "0,3", "--max-new-tokens", "2", "--mixer", "attention",
                        "--cache-dtype", "fp8", "--window", "3", "--sinks", "1"])
    text = capsys.readouterr().out
    assert "attention_impl: b200 (paged cache, fp8; seeded projections)" in text and "generated_tokens: 2" in text


def test_unknown_mixer_is_refused():
    from fastkernels_b200.decode_runner import DecodeRunner
    with pytest.raises(ValueError, match="mixer"):
        DecodeRunner([], synthetic_qwen36_spec(), mixer="deltanet")
