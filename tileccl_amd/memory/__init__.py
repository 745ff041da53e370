from tileccl_amd.memory.bump import BumpAllocator

__all__ = ["BumpAllocator", "SymmetricHeap", "free_collected"]


def __getattr__(name: str):
    if name == "SymmetricHeap":
        from tileccl_amd.memory.symmetric_heap import SymmetricHeap

        return SymmetricHeap
    if name == "free_collected":
        from tileccl_amd.memory.arena import free_collected

        return free_collected
    raise AttributeError(name)
