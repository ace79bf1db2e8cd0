"""tests/dist_shard_worker.py with FusedMuon in FusedAdamW's place (same arguments, same dump)."""
import dist_shard_worker as worker

_run = worker.run


def run(rank, world, port, args):
    import tossctr
    tossctr.FusedAdamW = tossctr.FusedMuon
    _run(rank, world, port, args)


if __name__ == "__main__":
    worker.run = run
    worker.main()
