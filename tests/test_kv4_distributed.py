"""The cache's format in the ranks' handshake, on Gloo CPU processes: a rank whose cache
holds its rows otherwise than the leader's must not start."""

import tempfile
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist

from tests.test_nebula_distributed import CFG, _spawn

pytestmark = [pytest.mark.distributed,
              pytest.mark.skipif(not (dist.is_available() and dist.is_gloo_available()), reason="no gloo")]


def _handshakes(rank, store):
    from forgeml_b200.nebula import DecoderConfig, Engine, EngineFailed, ParallelContext
    from tests.cpu_engine import CpuShardedDecoder

    torch.set_num_threads(1)
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2,
                            timeout=timedelta(seconds=20))
    ctx = ParallelContext.from_env(tp_size=2, pp_size=1, timeout_s=20)
    engine = Engine(DecoderConfig(**CFG), context=ctx, max_requests=4, decoder_factory=CpuShardedDecoder)
    for leader, worker in ((None, None), (4, 4), (4, None), (None, 4)):
        mine = worker if rank else leader
        if rank == 0 or leader == worker:
            engine._handshake(torch.float32, mine)
        else:
            with pytest.raises(EngineFailed, match="configuration differs"):
                engine._handshake(torch.float32, mine)
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_must_agree_on_the_cache_format():
    with tempfile.TemporaryDirectory() as d:
        procs = _spawn(_handshakes, (f"{d}/store",), 2, 60)
        assert [p.exitcode for p in procs.processes] == [0, 0]
