"""A device-side wait that runs out must end in an error status, not in a hang.

Every wait in the kernels (mbarrier or flag) has a time limit (`lucid_set_wait_limit_ns`, 2 s by default).
Here the limit is set to 0, which the kernels read as "do not wait": the first wait that is not satisfied at
once (the first tile load, at the latest) counts as expired, in every CTA.  The call must come back with a LucidKernelError that
names the kernel and the place, the GPU must stay usable, and a normal call on the same workspace afterwards
must give the right answer.  Nothing is made to fault: the kernels simply give up, wait out their copies in
flight, free their tensor memory and return.  The reference has no counterpart (its waits spin without limit,
forward_sub_fwd.py:541-544).

Collected late on purpose (file name), after the parity tests.
"""
import pytest
import torch

from oracle import lucid_oracle as orc

pytestmark = pytest.mark.gpu


def test_expired_wait_is_reported_and_the_next_call_is_fine():
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200._cabi import LucidKernelError
    from lucid_kernels_b200.cute import _forward_sub_fwd

    lib = _cabi.load()
    K, V, _ = orc.make_inputs(1, 8192, 1, dtype=torch.bfloat16, seed=81)
    Kc, Vc = K.cuda(), V.cuda()
    good = _forward_sub_fwd(Kc, Vc, check=True)
    torch.cuda.synchronize()
    try:
        lib.lucid_set_pair_solve(0)                   # the plain one-CTA-per-row-block path
        lib.lucid_set_wait_limit_ns(0)
        with pytest.raises(LucidKernelError) as err:
            _forward_sub_fwd(Kc, Vc, check=True)
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
        lib.lucid_set_pair_limits(8, 0)
    msg = str(err.value)
    assert "timed out" in msg or "never published" in msg or "left early" in msg, msg
    assert "kernel=" in msg and "row_block=" in msg
    torch.cuda.synchronize()
    # same workspace, default limit: the status words are cleared by the call and the result is right again
    again = _forward_sub_fwd(Kc, Vc, check=True)
    assert torch.equal(again, good)
    assert orc.rel_err(again, orc.forward_sub_blockwise(K, V)) < 0.01


@pytest.mark.parametrize("B,N,H,settings", [
    (1, 4096, 4, {}),                                                        # reverse solve with the upper dK sums, then the rest of dK
    (1, 4096, 4, dict(lucid_set_upper_in_solve=0)),                          # reverse solve, then dK over all tiles
    (1, 19072, 2, {}),                                                       # one launch, two items per row-block of dK
    (1, 38016, 1, dict(lucid_set_dk_split=0)),                               # one launch, one item per row-block
], ids=["upper", "separate", "fused-split", "fused"])
def test_a_backward_whose_waits_run_out_ends(B, N, H, settings):
    """Limits from none to about what the call needs, so that waits of all roles run out at all stages: every call comes
    back, and one that reports nothing is right, bit for bit.  (256 polls pass before a limit above 0 counts.)"""
    from lucid_kernels_b200 import _cabi
    from lucid_kernels_b200._cabi import LucidKernelError
    from lucid_kernels_b200.cute import _forward_sub_bwd_combined, _forward_sub_fwd

    lib = _cabi.load()
    K, V, G = (t.cuda() for t in orc.make_inputs(B, N, H, dtype=torch.bfloat16, seed=82))
    vp = _forward_sub_fwd(K, V, check=True)
    call = lambda: _forward_sub_bwd_combined(K, vp, G, use_diag_solve=True, check=True)
    ended = 0
    try:
        lib.lucid_set_pair_solve(0)
        for name, value in settings.items():
            getattr(lib, name)(value)
        good = call()
        for limit in (0, 1, 30_000, 100_000, 200_000, 400_000, 700_000, 1_000_000, 1_500_000):
            lib.lucid_set_wait_limit_ns(limit)
            for _ in range(3):
                try:
                    got = call()
                except LucidKernelError:
                    ended += 1
                else:
                    assert all(torch.equal(x, y) for x, y in zip(got, good)), limit
        assert ended > 0
        lib.lucid_set_wait_limit_ns(2_000_000_000)
        assert all(torch.equal(x, y) for x, y in zip(call(), good))
    finally:
        lib.lucid_set_wait_limit_ns(2_000_000_000)
        lib.lucid_set_pair_limits(8, 0)
        lib.lucid_set_upper_in_solve(1)
        lib.lucid_set_dk_split(1)
