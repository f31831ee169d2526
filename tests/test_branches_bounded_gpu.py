"""The error path of tree attention's bounded waits, run without any fault: a test build with a short limit and a flag that keeps the
loading thread from requesting anything lets every other wait run out. The kernel returns by itself with a code, ``gemm_tc_check``
raises, and the next ordinary launch is right: tensor memory was given back."""
import pytest
import torch

from dryft_challenge_htn_2026_b200.csrc import api
from test_branches_gpu import attend, tree_case

pytestmark = pytest.mark.gpu


def test_tree_attention_whose_loads_never_come_reports_and_the_next_one_is_right(monkeypatch):
    real = api._lib
    stall = lambda source, defines=None: real(source, dict(defines or {}, DK_TEST_STALL=1, DK_WAIT_CYCLES="4000000LL")
                                              if source == "attention_tree_tc.cu" else defines)
    monkeypatch.setattr(api, "_lib", stall)
    switch = lambda on: stall("attention_tree_tc.cu", {"HD": 128}).dk_test_stall(int(on))
    c = tree_case([200, 70], [9, 40], 8, 2, 128, torch.bfloat16, seed=1)
    assert switch(False) == 0
    good = attend(c)
    api.gemm_tc_check()
    try:
        assert switch(True) == 0
        attend(c)
        torch.cuda.synchronize()                      # the kernel came back by itself
        with pytest.raises(api.KernelError, match="attention_tree: a bounded wait.*2[1-3]"):
            api.gemm_tc_check()
    finally:
        switch(False)
    assert torch.equal(attend(c), good)
    api.gemm_tc_check()
