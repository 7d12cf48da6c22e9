"""CPU: what the log-probability entry points refuse, and the oracle's known answers."""
import ctypes
import math

import pytest
import torch

from nebulasd_b200 import _lib
from nebulasd_b200.logprobs import token_logprobs
from oracle.logprobs import token_logprobs as oracle

OK = 0


def _call(logits=4096, dtype=0, stride=100, vocab=100, rows=0, tokens=None, top=0, lp=None, rk=None, ent=None,
          ids=None, tops=None):
    return _lib.lib.neb_token_logprobs(logits, dtype, stride, vocab, rows, tokens, top, lp, rk, ent, ids, tops,
                                       None, None)


def test_no_rows_is_no_work():
    assert _call() == OK


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(vocab=0), dict(stride=-1), dict(top=-1), dict(top=33),
    dict(vocab=4, top=5), dict(rows=1, logits=None), dict(rows=1, tokens=64), dict(rows=1, lp=64),
    dict(rows=1, tokens=64, lp=64), dict(rows=1, tokens=64, rk=64), dict(rows=1, top=2), dict(rows=1, top=2, ids=64),
    dict(rows=1, logits=4097), dict(rows=1, dtype=2, logits=4098),
])
def test_the_c_entry_refuses(kw):
    assert _call(**kw) == _lib.NEB_ERR_INVALID
    assert _lib.lib.neb_last_error()


def test_rows_beyond_an_int_are_refused():
    assert _call(vocab=1 << 30) == OK
    assert _call(vocab=(1 << 30) + 1) == _lib.NEB_ERR_UNSUPPORTED


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((2, 10), dtype=torch.float16))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros((2, 10), dtype=torch.int32))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(10, dtype=torch.float16))


def test_oracle_known_answers():
    x = torch.tensor([[0.0, 0.0, 0.0, 0.0], [math.log(2.0), 0.0, -math.inf, -math.inf],
                      [1.0, math.nan, 2.0, math.inf]], dtype=torch.float64)
    lp, rk, ent, ids, tops = oracle(x, [3, 1, 0], 3)
    assert lp[:2] == pytest.approx([-math.log(4), -math.log(3)]) and math.isnan(lp[2])
    assert rk.tolist() == [1, 2, 4]
    assert ent[:2] == pytest.approx([math.log(4), math.log(3) - 2 / 3 * math.log(2)]) and math.isnan(ent[2])
    assert ids.tolist() == [[0, 1, 2], [0, 1, 2], [1, 3, 2]]
    assert tops[1].tolist() == pytest.approx([math.log(2 / 3), -math.log(3), -math.inf])
