"""-m gpu : the walk of every window class and stride in calls of several lengths, with many more tuples of capacity than tuples, so that
the walk moves them (integer outputs, exact against the oracle)."""
import numpy as np
import pytest
import torch

import cases

pytestmark = pytest.mark.gpu

# targets and frames whose band takes the window with that many states per lane, path stride 2 and 4 (window_max_tokens raised, so
# that the fast window is tried on paths of more than 64 targets)
SHAPES = {(1, 2): (32, 70), (2, 2): (75, 160), (3, 2): (110, 240), (4, 2): (188, 500), (6, 2): (240, 560), (8, 2): (380, 900),
          (1, 4): (18, 90), (2, 4): (40, 190), (3, 4): (60, 270), (4, 4): (90, 400), (6, 4): (140, 620), (8, 4): (200, 900)}


def batch(rw, stride, seed):
    rng = np.random.default_rng(seed)
    S0, T0 = SHAPES[rw, stride]
    lps, toks = [], []
    for k in range(9):
        S = S0 - k
        T = max(T0 - 3 * k, stride * S + 1)
        lp, tk, _ = cases.planted_case(rng, T, S, C=67, blank=66, peak=(9.0, 6.0, 3.0)[k % 3], sigma=1.0)
        lps.append(lp)
        toks.append(tk)
    return cases.pad_batch(lps, toks, 67, 66)


def aligned(lp, tk, T_len, S_len, dev, hint, seg_cap):
    from bournemouth_forced_aligner_amd import AlignmentUtils
    au = AlignmentUtils(66, 0, silence_anchors=0)
    au.viterbi_decoder.window_max_tokens = 4096
    return au.viterbi_decoder.align_batch(torch.from_numpy(lp).to(dev), torch.from_numpy(tk), T_len, S_len, anchor_pauses=False,
                                          seg_cap=seg_cap, class_mask=hint)


def check(ora, lp, tk, T_len, S_len, res):
    exp = ora.decode_alignments(lp, tk, T_len, S_len, ora.make_params(66, 0, 0, True, True, True, True), simple=False)
    assert (res.status.cpu().numpy() == exp["status"]).all()
    ph, idx, cnt, segs = (t.cpu().numpy() for t in (res.frame_phonemes, res.frame_phonemes_idx, res.seg_count, res.segs))
    for b in range(len(T_len)):
        T = int(T_len[b])
        np.testing.assert_array_equal(ph[b, :T], exp["frame_ph"][b, :T])
        np.testing.assert_array_equal(idx[b, :T], exp["frame_idx"][b, :T])
        assert cnt[b] == exp["seg_count"][b]
        np.testing.assert_array_equal(segs[b, :cnt[b]], exp["seg"][b, :cnt[b]])


@pytest.mark.parametrize("hint", [None, 0])
@pytest.mark.parametrize("rw,stride", sorted(SHAPES))
def test_tuples_of_every_window_class(ora, gpu_device, rw, stride, hint):
    lp, tk, T_len, S_len = batch(rw, stride, 10 * rw + stride)
    res = aligned(lp, tk, T_len, S_len, gpu_device, hint, lp.shape[1] + 1)
    torch.cuda.synchronize()
    check(ora, lp, tk, T_len, S_len, res)
