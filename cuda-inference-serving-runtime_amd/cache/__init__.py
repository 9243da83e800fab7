from .pages import FourBitNeed, KVNeed, StateNeed, OutOfPages, PagePool, CacheGroup
from .state import StateSlots
from .manager import CacheManager, Appended, pages_addressable, pages_that_fit
