"""Tensors whose memory is not what they show: negated views and storages that were given up are refused."""
import pytest
import torch

from test_learned_maps_record_nothing import CASES, calls


@pytest.mark.parametrize("i,name", CASES)
def test_pending_negations_are_refused(i, name):
    call, kw = list(calls())[i]
    kw[name] = torch._neg_view(kw[name])   # as z.conj().imag is
    assert kw[name].is_neg()
    with pytest.raises(ValueError, match="negation"):
        call(**kw)


@pytest.mark.parametrize("i,name", [(0, "initial_state"), (1, "d_final_state"), (2, "state"), (3, "state_out")])
def test_states_without_memory_are_refused(i, name):
    call, kw = list(calls())[i]
    kw[name].untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no memory"):
        call(**kw)
