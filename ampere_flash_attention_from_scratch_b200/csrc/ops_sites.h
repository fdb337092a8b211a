// ops_sites.h -- sites of the bounded waits of the kernel for many query rows over
// the 4-bit cache, behind those of the dense kernel (WaitSite).  Reported as
// AFA_DEV_TIMEOUT_BASE + site.
#pragma once

namespace afa100 {

enum WideSite : int {
  kSiteWideQ = 32,
  kSiteWideKFull = 33,
  kSiteWideVFull = 34,
  kSiteWideS = 35,
  kSiteWideP = 36,
  kSiteWidePv = 37,
  kSiteWideDrain = 38,
};

}  // namespace afa100
