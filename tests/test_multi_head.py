"""A tensor-parallel head in front of the vocabulary-sharded sampler on gloo ranks: VocabShardedSampler.sample_hidden
with a stand-in head (a product on the CPU over the rank's rows of the weights) and the host side's exchange, oracle
and result sharing in the place of the GPU's; every rank holds the tokens and states of the unsharded head."""
import os

import numpy as np
import pytest

from test_multi import _free_port

ROWS, VOCAB, K = 13, 1000, 24


def _case():
    from lrs import workloads as W
    rng = np.random.default_rng(21)
    p = np.zeros(ROWS, W.PARAMS_DTYPE)
    p["temperature"], p["top_k"], p["top_p"], p["repetition_penalty"], p["repeat_last_n"] = 0.8, 40, 0.95, 1.0, 64
    # (small whole numbers: every sum is exact, so that the shards' logits are the whole's bits)
    return (rng.integers(-3, 4, (ROWS, K)).astype(np.float32), rng.integers(-2, 3, (VOCAB, K)).astype(np.float32), p,
            np.arange(1, 2 * ROWS, 2, dtype=np.uint64), np.zeros((ROWS, 4), np.uint32), np.zeros(ROWS, np.uint32))


def _worker(rank, world, port, out_dir):
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    repo = os.path.dirname(here)
    for p in (os.path.join(repo, "llama.rs_b200"), os.path.join(repo, "oracle"), here):
        if p not in sys.path:
            sys.path.insert(0, p)
    import datetime

    import torch
    import torch.distributed as dist

    import oracle as O
    from lrs import sharded as S
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    try:
        hidden, weight, params, state, hist, hist_len = _case()

        class Head:
            device, vocab = torch.device("cuda:0"), VOCAB // world

            def logits(self, h):
                return h @ torch.from_numpy(weight[S.shard_columns(VOCAB, world, rank)]).t()

        class Sampler(S.VocabShardedSampler):
            def __init__(self):
                from lrs import BatchSampler
                self.rows, self.shard_n = ROWS, VOCAB // world
                self.bs = BatchSampler.__new__(BatchSampler)
                self.bs._h, self.bs.device = None, 0
                self.bs.check_rows = lambda rows, **buffers: None  # (they lie on the host here)

            def sample(self, shard, params, state, tokens, hist=None, hist_len=None, probs=None, status=None, stream=None):
                full = S.owner_exchange_host(shard.numpy(), ROWS)
                own = S.row_block(ROWS, world, rank)
                sl = slice(own.start, own.stop)
                tok, _, st = O.sample_batch(full, VOCAB, hist[sl], hist_len[sl], params[sl], state[sl], threads=1)
                res = S.share_rows_host(np.stack([tok.astype(np.uint64), st], axis=1), ROWS)
                tokens[:], state[:] = res.T

        vs, tokens = Sampler(), np.zeros(ROWS, np.uint64)
        vs.sample_hidden(Head(), torch.from_numpy(hidden), params, state, tokens, hist=hist, hist_len=hist_len)
        with pytest.raises(ValueError, match="hidden states are needed"):
            vs.sample_hidden(Head(), torch.from_numpy(hidden[1:]), params, state, tokens, hist=hist, hist_len=hist_len)
        np.save(os.path.join(out_dir, f"head_{rank}.npy"), np.stack([tokens, state]))
        dist.barrier()
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_a_sharded_head_gives_the_whole_heads_tokens(tmp_path, oracle, world):
    import torch.multiprocessing as mp
    mp.start_processes(_worker, args=(world, _free_port(), str(tmp_path)), nprocs=world, start_method="spawn")
    hidden, weight, params, state, hist, hist_len = _case()
    tok, _, st = oracle.sample_batch(hidden @ weight.T, VOCAB, hist, hist_len, params, state, threads=1)
    for r in range(world):
        got = np.load(tmp_path / f"head_{r}.npy")
        np.testing.assert_array_equal(got[0], tok.astype(np.uint64))
        np.testing.assert_array_equal(got[1], st)
