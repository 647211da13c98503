"""Edges of the decoding operators' contracts that need no GPU."""
import os
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nspeech_b200", "csrc")


@pytest.mark.parametrize("name", ["nq8_beam.cu", "nq8_cache.cu", "nq8_window_attention.cu", "nq8_window_attention.cuh",
                                  "nq8_window_attention_tc.cu", "nq8_gemv.cu"])
def test_decoding_kernels_read_by_plain_loads(name):
    """These kernels start before their predecessor has ended: what it writes must not go through the read-only path."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"__ldg|__ldcs|ld\.global\.nc|__restrict__", code)


@pytest.mark.parametrize("name,data", [("nq8_aux.cu", "x"), ("nq8_conv.cu", "x|cols"), ("nq8_qtiled.cu", r"xr|sx\d"), ("nq8_attention.cu", r"krel|p\.len|vrel"),
                                       ("nq8_encoder_kernels.cu", "mel|len0|len1|len|len_in|in|u|qkv|krel|x|src|row")])
def test_activations_and_lengths_are_read_by_plain_loads(name, data):
    """The same for the other kernels; weights, which no kernel changes, may take the read-only path."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(rf"const \w+ \*__restrict__ (?:{data})\b", code)
    assert not re.findall(rf"__ldg\((?:reinterpret_cast<[^>]*>\()?(?:{data})\b", code)


def test_one_beam_s_rows_may_lie_any_distance_apart():
    """Greedy decoding over a padded lm_head: with one beam its own stride means nothing.  The refusal left is the host tensor's."""
    from nspeech_b200.beam import beam_select
    from nspeech_b200.fast_matmul import MatMulError
    padded, scores = torch.zeros((4, 100)), torch.zeros((4, 1))
    for logits in (padded[:, :90].unsqueeze(1), torch.zeros((4, 3, 90))[:, -1:], torch.zeros((4, 1, 90))):
        with pytest.raises(MatMulError, match="CUDA"):
            beam_select(logits, scores)
    with pytest.raises(MatMulError, match="evenly spaced"):
        beam_select(torch.zeros((4, 3, 90))[:, :2], torch.zeros((4, 2)))


def test_python_refuses_what_wants_a_gradient_or_stands_for_other_values():
    from nspeech_b200.attention import window_attention
    from nspeech_b200.beam import beam_reorder, beam_select
    from nspeech_b200.fast_matmul import MatMulError
    q, x, s, parents = torch.zeros((4, 2, 64)), torch.zeros((1, 2, 9)), torch.zeros((1, 2)), torch.zeros(4, dtype=torch.int32)
    calls = [lambda t: window_attention(t(q), q, q), lambda t: window_attention(q, t(q), q), lambda t: window_attention(q, q, t(q)),
             lambda t: window_attention(q, q, q, out=t(q)), lambda t: beam_select(t(x), s), lambda t: beam_select(x, t(s))]
    learns = [lambda t: t.clone().requires_grad_(), lambda t: t.clone().requires_grad_() * 1]
    for call in calls:
        for how in learns:
            with pytest.raises(MatMulError, match="gradient"):
                call(how)
            with torch.no_grad(), pytest.raises(MatMulError, match="CUDA"):  # as far as any host tensor comes
                call(how)
        with pytest.raises(MatMulError, match="negated"):
            call(torch._neg_view)
    with pytest.raises(MatMulError, match="negated"):
        beam_reorder([q], torch._neg_view(parents))


def test_python_refuses_outputs_that_overlap():
    from nspeech_b200.attention import window_attention
    from nspeech_b200.beam import beam_select
    from nspeech_b200.fast_matmul import MatMulError
    whole = torch.zeros((12, 2, 64))
    q, k, v, out = whole[:4], whole[4:8], whole[8:], torch.zeros((4, 2, 64))
    for bad in (k, v, whole[2:6], whole[1:5], torch.zeros((4, 1, 64)).expand(4, 2, 64), torch.zeros((1, 2, 64)).expand(4, 2, 64)):
        with pytest.raises(MatMulError, match="overlaps"):
            window_attention(q, k, v, out=bad)
    for good in (out, q):  # rows are read before their places are written
        with pytest.raises(MatMulError, match="CUDA"):
            window_attention(q, k, v, out=good)
    x, s, fin = torch.zeros((1, 2, 9)), torch.zeros((1, 2)), torch.zeros((1, 2), dtype=torch.bool)
    a, b = torch.zeros((1, 2), dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    for bad in ((s, a, a, fin), (x[0, :1, :2], a, b, fin), (s, s.view(torch.int32), b, fin)):
        with pytest.raises(MatMulError, match="overlaps"):
            beam_select(x, s, fin, 1, out=bad)
    with pytest.raises(MatMulError, match="CUDA"):
        beam_select(x, s, fin, 1, out=(s, a, b, fin))


def test_the_library_builds_without_python():
    """The C ABI's users have nvcc and g++: by itself `make` asks for nothing of Python or torch."""
    def commands(*targets):
        r = subprocess.run(["make", "-n", "-B", "-C", CSRC, *targets], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        return r.stdout
    assert "libnq8.so" in commands() and not re.search("torch|nq8_py|python", commands())
    assert "nq8_py.so" in commands("python") and "libnq8.so" in commands("python")
