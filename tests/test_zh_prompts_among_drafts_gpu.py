"""Slots that bring prompts beside slots with drafted tokens: u_accept of -1 lets every token of a prompt stand, whatever the probabilities."""
import numpy as np
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("vocab", [97, 20001])
def test_prompts_stand(vocab, with_q):
    from flashrt_b200 import flash_rt_kernels as fvk
    rng = np.random.default_rng(vocab + with_q)
    rows = [5, 300, 1, 0, 33, 4, 64]                                 # the second, fifth and last are prompts
    prompts = (1, 4, 6)
    cu = np.concatenate([[0], np.cumsum(rows)]).tolist()
    n = cu[-1]
    p = rng.random((n, vocab), dtype=np.float32) * (rng.random((n, vocab)) < 0.1)
    p[np.arange(n), rng.integers(0, vocab, n)] += 1
    tokens = rng.integers(0, vocab, n).astype(np.int32)
    u, v = rng.random(n, dtype=np.float32), rng.random(len(rows), dtype=np.float32)
    q = np.maximum(p, 0.25).astype(np.float32) if with_q else None
    for s in prompts:
        u[cu[s]:cu[s + 1]] = -1
        for t in range(cu[s], cu[s + 1] - 1):
            p[t, tokens[t + 1]] = 0                                  # the target would never say so
    lens = rng.integers(400, 500, len(rows)).astype(np.int32)
    d = {k: torch.from_numpy(np.asarray(x)).cuda() for k, x in dict(p=p, tokens=tokens, cu=np.asarray(cu, np.int32), lens=lens, u=u, v=v).items()}
    dq = torch.from_numpy(q).cuda() if with_q else None
    out, accepted, kept = (torch.full((k,), -9, dtype=I32, device="cuda") for k in (n, len(rows), len(rows)))
    fvk.verify_drafts(d["p"].data_ptr(), dq.data_ptr() if with_q else 0, d["tokens"].data_ptr(), d["cu"].data_ptr(), d["lens"].data_ptr(),
                      d["u"].data_ptr(), d["v"].data_ptr(), out.data_ptr(), accepted.data_ptr(), kept.data_ptr(), n, len(rows), vocab,
                      torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    want, acc, stay = R.verify(p, q, tokens.tolist(), cu, lens.tolist(), u, v)
    assert out.tolist() == want and accepted.tolist() == acc and kept.tolist() == stay
    for s in prompts:
        assert acc[s] == rows[s] - 1 and stay[s] == lens[s] and out[cu[s]:cu[s + 1] - 1].tolist() == tokens[cu[s] + 1:cu[s + 1]].tolist()
